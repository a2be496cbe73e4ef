// AdamW over many tensors in one launch, moments held in f32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,  p = p - (lr wd p + lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps))
//
// Bound by HBM: 28 bytes per element with f32 gradients and moments, 16 with 8-bit moments, each touched
// once.  The tensors' pointers travel as kernel arguments (no table in device memory to fill, so a launch
// can be captured into a graph); a workgroup owns 4096 consecutive elements of one tensor and finds it
// with one comparison per lane.
//
// 8-bit moments.  256 consecutive elements of a tensor share one exponent byte E, the f32 exponent of their
// largest magnitude (one more when that lies above 1.875 times its power of two, so that rounding up never
// leaves the range).  The codes are f32 bit patterns cut to three mantissa bits, counted from the top of the
// block: bits = (code + 8 E - 120) << 20 for the first moment (a sign bit and 7 bits of magnitude: 15 binades
// below the largest), bits = (code + 8 E - 248) << 20 for the second (8 bits: 31 binades); code 0 is zero.
// Integer shifts alone convert, exactly, and every value is exact in bf16.  A moment moves by less than one
// code per step (the second by a thousandth of its value), so rounding to nearest would hold it in place
// for ever: codes are rounded stochastically, with 16 bits of an integer hash of (seed, step, tensor,
// element), which keeps the moments unbiased and a run reproducible.  A second moment is never rounded to
// zero (its square root divides): one below the smallest code, 2^-31 of the block's largest, is raised to it.  The update of p uses the moments before they are rounded.
//
// Measured on 68.3 M elements in 40 tensors (a copy of 1 GiB runs at 5.05 TB/s on the same card): f32 gradients and moments 360 us,
// 1.91 GB, 5.3 TB/s; bf16 gradients and 8-bit moments 202 us, 0.96 GB, 4.7 TB/s, and their values as bf16 (adamw_moments) 82 us,
// 0.41 GB, 5.0 TB/s.  16 tensors with 2.8 M elements: 13 us, and the launch around it costs the host more.
#include "sf_common.h"
#include <float.h>
#include "../../include/sfhip.h"

namespace {

constexpr int NT = 256;
constexpr int CHUNK = 4096;        // elements of a workgroup: 16 per thread
constexpr int BLOCK = SF_ADAMW_BLOCK;
constexpr long long MAX_GROUPS = (1 << 24) - 1;     // workgroups of one launch: less than 2^32 threads
constexpr long long MAX_ELEMENTS = MAX_GROUPS * CHUNK;
static_assert(BLOCK == 8 * 32 && CHUNK % (8 * NT) == 0, "32 lanes hold a block of moments");

struct Tensor {
    float* p;
    const void* g;
    void* m;
    void* v;
    unsigned char* me;
    unsigned char* ve;
    bf16* shadow;
    long long n;
    float lr, decay;               // decay = lr * weight decay
    int step_offset;
    int ordinal;                   // position in the call's list (enters the hash)
    int g_bf16;
    int first;                     // first workgroup
};
struct Hyper { double beta1, beta2; float eps, grad_scale; unsigned seed_lo, seed_hi; int count; };
// tensors of one launch: as many as 4 KB of kernel arguments hold beside two pointers and the 256 bytes that the compiler adds
constexpr int MAX_TENSORS = (4096 - 256 - 16 - (int)sizeof(Hyper)) / (int)sizeof(Tensor);
static_assert(MAX_TENSORS <= 64, "a lane for each");
struct Table { Tensor t[MAX_TENSORS]; };

// V elements at an address aligned to one element only: the hardware serves wide global accesses at any element alignment
template <typename T, int V> struct __attribute__((packed, aligned(sizeof(T)))) Some { T e[V]; };

// WHOLE: the workgroup's elements all exist, otherwise the first `have` of the V do (the others read as zero)
template <bool WHOLE, int V, typename T> __device__ __forceinline__ Some<T, V> load_some(const T* p, int have) {
    Some<T, V> r{};
    if constexpr (WHOLE) {
        r = *reinterpret_cast<const Some<T, V>*>(p);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < have) r.e[j] = p[j];
    }
    return r;
}
template <bool WHOLE, int V, typename T> __device__ __forceinline__ void store_some(T* p, int have, const Some<T, V>& v) {
    if constexpr (WHOLE) {
        *reinterpret_cast<Some<T, V>*>(p) = v;
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < have) p[j] = v.e[j];
    }
}

// b^t by squaring (t >= 1)
__device__ __forceinline__ double power(double b, int t) {
    double r = 1.0;
    for (; t > 0; t >>= 1) {
        if (t & 1) r *= b;
        b *= b;
    }
    return r;
}

__host__ __device__ __forceinline__ unsigned mix(unsigned x) {
    x ^= x >> 16;
    x *= 0x6A09E667u;
    x ^= x >> 15;
    x *= 0xBB67AE85u;
    return x ^ (x >> 16);
}

// largest value among the 32 lanes of a half wave, in all of them: rotations within 16 lanes, then the two sixteens
// change places (vector instructions only, no trip through LDS)
__device__ __forceinline__ unsigned half_wave_max(unsigned v) {
    const auto turned = [](unsigned x, auto ctrl) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, ctrl.value, 0xf, 0xf, false); };
    unsigned t = turned(v, std::integral_constant<int, 0x128>{});      // row_ror:8
    v = v > t ? v : t;
    t = turned(v, std::integral_constant<int, 0x124>{});
    v = v > t ? v : t;
    t = turned(v, std::integral_constant<int, 0x122>{});
    v = v > t ? v : t;
    t = turned(v, std::integral_constant<int, 0x121>{});
    v = v > t ? v : t;
    const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return s[0] > s[1] ? s[0] : s[1];
}

// f32 value of a code under block exponent e; SIGNED: first moment
template <bool SIGNED> __device__ __forceinline__ float decode(unsigned c, int e) {
    const unsigned low = SIGNED ? c & 127u : c;
    const unsigned bits = (low + 8u * (unsigned)e - (SIGNED ? 120u : 248u)) << 20;
    return low ? __uint_as_float(SIGNED ? bits | ((c & 128u) << 24) : bits) : 0.f;
}
// block exponent for the largest magnitude (as f32 bits); the lower bound keeps every code a normal f32
template <bool SIGNED> __device__ __forceinline__ int block_exponent(unsigned largest) {
    const unsigned e = (largest + 0xFFFFFu) >> 23;
    const unsigned least = SIGNED ? 16u : 32u;
    return (int)(e < least ? least : e > 255u ? 255u : e);
}
// code of x under block exponent e, rounded up with probability (distance to the code below) / (code spacing)
template <bool SIGNED> __device__ __forceinline__ unsigned encode(float x, int e, unsigned r16) {
    const unsigned bits = __float_as_uint(x) & 0x7FFFFFFFu;
    const unsigned base = 8u * (unsigned)e - (SIGNED ? 120u : 248u);
    const unsigned top = SIGNED ? 127u : 255u;
    const unsigned least = (base + 1u) << 20;
    unsigned c = ((bits + (r16 << 4)) >> 20) - base;
    c = c > top ? top : c;
    if (bits < least) {
        if (SIGNED) c = __uint_as_float(bits) > (float)r16 * (1.f / 65536.f) * __uint_as_float(least) ? 1u : 0u;
        else c = bits ? 1u : 0u;
    }
    return SIGNED ? c | ((__float_as_uint(x) >> 31) << 7) : c;
}

// the tensor that workgroup `bid` works on: lanes compare, the last first <= bid wins
__device__ __forceinline__ int tensor_of(const Table& tab, int count, int bid) {
    const int lane = threadIdx.x & 63;
    const bool before = lane < count && tab.t[lane < count ? lane : 0].first <= bid;
    return __builtin_amdgcn_readfirstlane(__popcll(__ballot(before)) - 1);
}

// One workgroup's 4096 elements.  BITS 32: a thread takes 4 consecutive elements at a time; BITS 8: 8, so that 32 lanes
// hold a block of moments.
template <int BITS, bool WHOLE, typename G>
__device__ __forceinline__ void adamw_chunk(const Tensor& T, const Hyper& h, long long c0, int t_all) {
    constexpr int V = BITS == 32 ? 4 : 8, U = CHUNK / (V * NT);
    const float b1 = (float)h.beta1, b2 = (float)h.beta2, a1 = (float)(1.0 - h.beta1), a2 = (float)(1.0 - h.beta2);
    long long at[U];
    int have[U];
    Some<float, V> p[U], m[U], v[U];
    Some<G, V> g[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        at[u] = c0 + u * (V * NT) + threadIdx.x * V;
        const long long left = T.n - at[u];
        have[u] = left >= V ? V : left > 0 ? (int)left : 0;
        g[u] = load_some<WHOLE, V>((const G*)T.g + at[u], have[u]);
        p[u] = load_some<WHOLE, V>(T.p + at[u], have[u]);
    }
    if constexpr (BITS == 32) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            m[u] = load_some<WHOLE, V>((const float*)T.m + at[u], have[u]);
            v[u] = load_some<WHOLE, V>((const float*)T.v + at[u], have[u]);
        }
    } else {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const auto cm = load_some<WHOLE, V>((const unsigned char*)T.m + at[u], have[u]);
            const auto cv = load_some<WHOLE, V>((const unsigned char*)T.v + at[u], have[u]);
            const int em = WHOLE || have[u] ? T.me[at[u] / BLOCK] : 16, ev = WHOLE || have[u] ? T.ve[at[u] / BLOCK] : 32;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                m[u].e[j] = decode<true>(cm.e[j], em);
                v[u].e[j] = decode<false>(cv.e[j], ev);
            }
        }
    }
    const int t = max(t_all + T.step_offset, 1);
    const float step = (float)((double)T.lr / (1.0 - power(h.beta1, t)));
    const float root = (float)(1.0 / sqrt(1.0 - power(h.beta2, t)));
    unsigned key = 0;
    if constexpr (BITS == 8) key = mix(mix((h.seed_lo + (unsigned)t_all * 0x9E3779B1u) ^ h.seed_hi) + (unsigned)T.ordinal * 0x85EBCA6Bu);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        unsigned mm = 0, mv = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float gs = to_f32(g[u].e[j]) * h.grad_scale;
            m[u].e[j] = b1 * m[u].e[j] + a1 * gs;
            v[u].e[j] = b2 * v[u].e[j] + a2 * gs * gs;
            // (decay and step are added up before the one rounding into p: a factor 1 - decay would lose a decay below 2^-25.  The
            // product takes the largest finite value for an infinite one, which stays infinite so.)
            const float finite = fminf(fmaxf(p[u].e[j], -FLT_MAX), FLT_MAX);
            p[u].e[j] -= fmaf(T.decay, finite, step * (m[u].e[j] / (sqrtf(v[u].e[j]) * root + h.eps)));
            // (elements behind the tensor's end hold zero: nothing was loaded)
            const unsigned bm = __float_as_uint(m[u].e[j]) & 0x7FFFFFFFu, bv = __float_as_uint(v[u].e[j]) & 0x7FFFFFFFu;
            mm = mm > bm ? mm : bm;
            mv = mv > bv ? mv : bv;
        }
        store_some<WHOLE, V>(T.p + at[u], have[u], p[u]);
        if (T.shadow) {
            Some<bf16, V> s;
#pragma unroll
            for (int j = 0; j < V; ++j) s.e[j] = (bf16)p[u].e[j];
            store_some<WHOLE, V>(T.shadow + at[u], have[u], s);
        }
        if constexpr (BITS == 32) {
            store_some<WHOLE, V>((float*)T.m + at[u], have[u], m[u]);
            store_some<WHOLE, V>((float*)T.v + at[u], have[u], v[u]);
        } else {
            const int em = block_exponent<true>(half_wave_max(mm)), ev = block_exponent<false>(half_wave_max(mv));
            Some<unsigned char, V> cm, cv;
            const unsigned base = (unsigned)at[u] * 0x9E3779B1u + (unsigned)(at[u] >> 32) * 0xC2B2AE35u + key;
#pragma unroll
            for (int j = 0; j < V; ++j) {       // (the upper half of the index is the same for all: V divides 2^32)
                const unsigned r = mix(base + (unsigned)j * 0x9E3779B1u);
                cm.e[j] = (unsigned char)encode<true>(m[u].e[j], em, r >> 16);
                cv.e[j] = (unsigned char)encode<false>(v[u].e[j], ev, r & 0xFFFFu);
            }
            store_some<WHOLE, V>((unsigned char*)T.m + at[u], have[u], cm);
            store_some<WHOLE, V>((unsigned char*)T.v + at[u], have[u], cv);
            if ((threadIdx.x & 31) == 0 && (WHOLE || have[u])) {
                T.me[at[u] / BLOCK] = (unsigned char)em;
                T.ve[at[u] / BLOCK] = (unsigned char)ev;
            }
        }
    }
}

template <int BITS>
__global__ __launch_bounds__(NT) void adamw_kernel(Table tab, Hyper h, const int* __restrict__ state,
                                                   const int* __restrict__ found_inf) {
    if (found_inf && found_inf[0] != 0) return;
    const Tensor& T = tab.t[tensor_of(tab, h.count, blockIdx.x)];
    const long long c0 = (long long)(blockIdx.x - T.first) * CHUNK;
    const int t_all = state[0];
    const bool whole = c0 + CHUNK <= T.n;
    if (T.g_bf16) {
        if (whole) adamw_chunk<BITS, true, bf16>(T, h, c0, t_all);
        else adamw_chunk<BITS, false, bf16>(T, h, c0, t_all);
    } else {
        if (whole) adamw_chunk<BITS, true, float>(T, h, c0, t_all);
        else adamw_chunk<BITS, false, float>(T, h, c0, t_all);
    }
}

// bf16 values of 8-bit moments (exact); T.p and T.shadow hold the two outputs
template <bool WHOLE> __device__ __forceinline__ void moments_chunk(const Tensor& T, long long c0) {
    constexpr int V = 8, U = CHUNK / (V * NT);
    long long at[U];
    int have[U], em[U], ev[U];
    Some<unsigned char, V> cm[U], cv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        at[u] = c0 + u * (V * NT) + threadIdx.x * V;
        const long long left = T.n - at[u];
        have[u] = left >= V ? V : left > 0 ? (int)left : 0;
        cm[u] = load_some<WHOLE, V>((const unsigned char*)T.m + at[u], have[u]);
        cv[u] = load_some<WHOLE, V>((const unsigned char*)T.v + at[u], have[u]);
        em[u] = WHOLE || have[u] ? T.me[at[u] / BLOCK] : 16;
        ev[u] = WHOLE || have[u] ? T.ve[at[u] / BLOCK] : 32;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        Some<bf16, V> m, v;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            m.e[j] = (bf16)decode<true>(cm[u].e[j], em[u]);
            v.e[j] = (bf16)decode<false>(cv[u].e[j], ev[u]);
        }
        store_some<WHOLE, V>((bf16*)T.p + at[u], have[u], m);
        store_some<WHOLE, V>(T.shadow + at[u], have[u], v);
    }
}
__global__ __launch_bounds__(NT) void adamw_moments_kernel(Table tab, int count) {
    const Tensor& T = tab.t[tensor_of(tab, count, blockIdx.x)];
    const long long c0 = (long long)(blockIdx.x - T.first) * CHUNK;
    if (c0 + CHUNK <= T.n) moments_chunk<true>(T, c0);
    else moments_chunk<false>(T, c0);
}

// splits the list into launches of at most MAX_TENSORS non-empty tensors and MAX_GROUPS workgroups
template <typename F, typename L> int over_tensors(int count, const long long* n, F&& fill, L&& launch) {
    Table tab;
    int used = 0;
    long long groups = 0;
    for (int i = 0; i <= count; ++i) {
        const long long need = i < count ? (n[i] + CHUNK - 1) / CHUNK : 0;
        if (used && (i == count || used == MAX_TENSORS || groups + need > MAX_GROUPS)) {
            launch(tab, used, (int)groups);
            used = 0;
            groups = 0;
        }
        if (i < count && n[i] > 0) {
            fill(tab.t[used], i);
            tab.t[used].first = (int)groups;
            groups += need;
            ++used;
        }
    }
    return SF_OK;
}

}  // namespace

extern "C" int sf_adamw_step(int count, float* const* p, const void* const* g, void* const* m, void* const* v,
                             unsigned char* const* m_exp, unsigned char* const* v_exp, void* const* shadow_bf16,
                             const long long* n, const double* lr, const double* weight_decay, const int* g_dtype,
                             const int* step_offset, int state_bits, double beta1, double beta2, float eps, float grad_scale,
                             unsigned long long seed, const int* state, const int* found_inf, void* stream) {
    SF_REQUIRE(count >= 0 && p && g && m && v && n && lr && weight_decay && g_dtype && state, "sf_adamw_step: null argument");
    SF_REQUIRE(state_bits == 32 || state_bits == 8, "sf_adamw_step: moments are held in 32 or 8 bits, not %d", state_bits);
    SF_REQUIRE(state_bits == 32 || (m_exp && v_exp), "sf_adamw_step: 8-bit moments need their block exponents");
    SF_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, "sf_adamw_step: betas must lie in [0, 1)");
    SF_REQUIRE(eps >= 0.f, "sf_adamw_step: eps must not be negative");
    for (int i = 0; i < count; ++i) {
        SF_REQUIRE(n[i] >= 0 && n[i] <= MAX_ELEMENTS, "sf_adamw_step: tensor %d has %lld elements", i, n[i]);
        SF_REQUIRE(n[i] == 0 || (p[i] && g[i] && m[i] && v[i]), "sf_adamw_step: tensor %d has a null pointer", i);
        SF_REQUIRE(n[i] == 0 || state_bits == 32 || (m_exp[i] && v_exp[i]), "sf_adamw_step: tensor %d lacks its exponents", i);
        SF_REQUIRE(g_dtype[i] == SF_F32 || g_dtype[i] == SF_BF16, "sf_adamw_step: tensor %d has gradient dtype %d", i, g_dtype[i]);
        SF_REQUIRE(!step_offset || step_offset[i] <= 0, "sf_adamw_step: step offsets are not positive");
    }
    Hyper h{beta1, beta2, eps, grad_scale, (unsigned)seed, (unsigned)(seed >> 32), 0};
    auto fill = [&](Tensor& t, int i) {
        t = Tensor{p[i], g[i], m[i], v[i], state_bits == 8 ? m_exp[i] : nullptr, state_bits == 8 ? v_exp[i] : nullptr,
                   shadow_bf16 ? (bf16*)shadow_bf16[i] : nullptr, n[i], (float)lr[i], (float)(lr[i] * weight_decay[i]),
                   step_offset ? step_offset[i] : 0, i, g_dtype[i] == SF_BF16, 0};
    };
    auto launch = [&](const Table& tab, int used, int groups) {
        h.count = used;
        if (state_bits == 32)
            hipLaunchKernelGGL((adamw_kernel<32>), dim3(groups), dim3(NT), 0, (hipStream_t)stream, tab, h, state, found_inf);
        else
            hipLaunchKernelGGL((adamw_kernel<8>), dim3(groups), dim3(NT), 0, (hipStream_t)stream, tab, h, state, found_inf);
    };
    over_tensors(count, n, fill, launch);
    SF_LAUNCH_CHECK("sf_adamw_step");
    return SF_OK;
}

extern "C" int sf_adamw_moments(int count, const void* const* m, const void* const* v, const unsigned char* const* m_exp,
                                const unsigned char* const* v_exp, void* const* m_bf16, void* const* v_bf16,
                                const long long* n, void* stream) {
    SF_REQUIRE(count >= 0 && m && v && m_exp && v_exp && m_bf16 && v_bf16 && n, "sf_adamw_moments: null argument");
    for (int i = 0; i < count; ++i) {
        SF_REQUIRE(n[i] >= 0 && n[i] <= MAX_ELEMENTS, "sf_adamw_moments: tensor %d has %lld elements", i, n[i]);
        SF_REQUIRE(n[i] == 0 || (m[i] && v[i] && m_exp[i] && v_exp[i] && m_bf16[i] && v_bf16[i]),
                   "sf_adamw_moments: tensor %d has a null pointer", i);
    }
    auto fill = [&](Tensor& t, int i) {
        t = Tensor{(float*)m_bf16[i], nullptr, (void*)m[i], (void*)v[i], (unsigned char*)m_exp[i], (unsigned char*)v_exp[i],
                   (bf16*)v_bf16[i], n[i], 0.f, 0.f, 0, i, 0, 0};
    };
    auto launch = [&](const Table& tab, int used, int groups) {
        hipLaunchKernelGGL(adamw_moments_kernel, dim3(groups), dim3(NT), 0, (hipStream_t)stream, tab, used);
    };
    over_tensors(count, n, fill, launch);
    SF_LAUNCH_CHECK("sf_adamw_moments");
    return SF_OK;
}
