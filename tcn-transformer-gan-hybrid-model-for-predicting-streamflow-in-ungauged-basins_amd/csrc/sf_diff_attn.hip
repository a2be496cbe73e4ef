// Differential attention, forward and backward.
//
//   per query head:  P_i = softmax(scale q_i k_i^T)  (i = 1, 2: the two halves of the head),  O_i = P_i v,
//   o = O_1 - lam O_2 = (P_1 - lam P_2) v
//   dv = (P_1 - lam P_2)^T do,   dP = do v^T,   delta_i = rowsum(P_i dP) = do . O_i,
//   dS_1 = P_1 (dP - delta_1),  dS_2 = -lam P_2 (dP - delta_2),  dq_i = scale dS_i k_i,  dk_i = scale dS_i^T q_i,
//   dlam = -sum delta_2
//
// The score matrices never exist in memory: tiles of 32 keys x 32 queries live in registers and the softmax runs
// online (running maximum and sum per row and map, f32; exponents in base 2).  All products are 32 x 32
// matrix instructions with f32 accumulation; probabilities and score gradients are rounded to the inputs' type to
// enter the second product (bf16: half a step of 2^-8 of each probability, the size of the inputs' own
// rounding).  The f32 form runs through the same code with f32 matrix instructions and rounds nothing.
//
// Layout.  Heads are [.., 2, d] rows (v and o: [.., 2 d], treated as two halves as well), d <= 64 a multiple of 8,
// padded to DP = 16, 32 or 64 columns per half inside a tile.  A tile in LDS is [row][2 DP], its 16-byte pieces
// XORed with a function of the row (Tile::swz) so that both ways of reading it spread over the banks: 32 rows at one
// piece (an operand whose reduction axis is the columns) and 4 x 4 rows at 32 columns (reduction over the rows,
// through the transposing LDS read).  Tiles arrive by buffer loads that write LDS directly; pieces outside
// a sample's rows or a head's columns are out of the buffer's range and arrive as zeros, so keys
// behind a sample's length are never read.  Accumulators hold [reduction-free axis of the second product] x
// [query or key], so that the query's (key's) softmax state and scale are one register per lane and the
// probabilities leave the first product in the very registers the second one reads (the reduction axis is permuted
// the same way in both of its operands).
#include "sf_common.h"
#include "../../include/sfhip.h"

namespace {

typedef __attribute__((address_space(3))) char* lds_ptr;
typedef bf16x4 __attribute__((address_space(3)))* lds_bf16x4;

// ---- one operand row piece: 8 values along the reduction axis
template <typename T> struct Frag;
template <> struct Frag<bf16> { bf16x8 v; };
template <> struct Frag<float> { float v[8]; };

__device__ __forceinline__ f32x16 mma(const Frag<bf16>& a, const Frag<bf16>& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(const Frag<float>& a, const Frag<float>& b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[j], b.v[j], c, 0, 0, 0);
    return c;
}
// 8 accumulator values (rows 4 h .. 4 h + 3 and 8 + 4 h .. of a 16-row step) as an operand of the next product
__device__ __forceinline__ void pack(Frag<bf16>& f, const float* x) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f.v[j] = (bf16)x[j];
}
__device__ __forceinline__ void pack(Frag<float>& f, const float* x) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f.v[j] = x[j];
}
__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}
// row of accumulator register r of a lane in half h = lane / 32
__device__ __forceinline__ constexpr int acc_row(int r, int h) { return 8 * (r / 4) + 4 * h + (r % 4); }

// ---- tiles in LDS
template <typename T, int DP> struct Tile {
    static constexpr int EPC = 16 / (int)sizeof(T);       // elements per 16-byte piece
    static constexpr int NCH = 2 * DP / EPC;              // pieces per row
    static constexpr int ROWB = NCH * 16;
    static constexpr int BITS = NCH >= 16 ? 4 : NCH == 8 ? 3 : 2;
    static constexpr int SHIFT = 4 - BITS;                // rows that share a 256-byte window
    // XOR of a row's pieces: the upper bits spread 4-row groups over piece pairs, the lowest bit the two halves of 16 rows
    static __device__ __forceinline__ int swz(int row) {
        const int s = (row & 15) >> SHIFT;
        return ((s & ((1 << (BITS - 1)) - 1)) << 1) | ((s >> (BITS - 1)) & 1);
    }
    // 8 columns from col (a multiple of 8) of one row
    static __device__ __forceinline__ Frag<T> row_piece(const char* t, int row, int col) {
        Frag<T> f;
        if constexpr (sizeof(T) == 2) {
            f.v = *reinterpret_cast<const bf16x8*>(t + row * ROWB + (((col >> 3) ^ swz(row)) << 4));
        } else {
            const int c = col >> 2;
            const float4 lo = *reinterpret_cast<const float4*>(t + row * ROWB + ((c ^ swz(row)) << 4));
            const float4 hi = *reinterpret_cast<const float4*>(t + row * ROWB + (((c + 1) ^ swz(row)) << 4));
            f.v[0] = lo.x; f.v[1] = lo.y; f.v[2] = lo.z; f.v[3] = lo.w;
            f.v[4] = hi.x; f.v[5] = hi.y; f.v[6] = hi.z; f.v[7] = hi.w;
        }
        return f;
    }
    // column col0 + lane % 32 of rows row0 + acc_row(0..7, lane / 32): the reduction axis is the rows, in the order the
    // accumulators hold them.  row0 a multiple of 16, col0 of 32.
    static __device__ __forceinline__ Frag<T> col_piece(const char* t, int row0, int col0, int lane) {
        const int h = lane >> 5;
        Frag<T> f;
        if constexpr (sizeof(T) == 2) {
            const int i = lane & 15, row = row0 + 4 * h + (i >> 2), col = col0 + 16 * ((lane >> 4) & 1) + 4 * (i & 3);
            const char* lo = t + row * ROWB + (((col >> 3) ^ swz(row)) << 4) + (col & 7) * 2;
            const char* hi = t + (row + 8) * ROWB + (((col >> 3) ^ swz(row + 8)) << 4) + (col & 7) * 2;
            const bf16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4)(lo));
            const bf16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4)(hi));
#pragma unroll
            for (int j = 0; j < 4; ++j) { f.v[j] = a[j]; f.v[4 + j] = b[j]; }
        } else {
            const int col = col0 + (lane & 31);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int row = row0 + acc_row(j, h);
                f.v[j] = *reinterpret_cast<const float*>(t + row * ROWB + (((col >> 2) ^ swz(row)) << 4) + (col & 3) * 4);
            }
        }
        return f;
    }
};

// 64 lanes x 16 bytes from the buffer's byte offsets `off` to LDS from `dst` on (uniform); zeros where the offset lies outside
// the buffer.  (Not in a template: in one, the host pass drops the launch stubs of every kernel that uses the builtin.)
__device__ __forceinline__ void copy_piece(__amdgpu_buffer_rsrc_t rs, char* dst, int off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr)dst, 16, off, 0, 0, 0);
}

// Copies ROWS rows of a [.., 2, d] array into a tile, NW waves together.  The byte offsets of a thread's pieces do not
// change from tile to tile; the tile's first row enters through the buffer's base address (64 bits).
template <typename T, int DP, int ROWS, int NW> struct Copy {
    using L = Tile<T, DP>;
    static constexpr int PIECES = ROWS * L::NCH;
    static constexpr int JOBS = (PIECES + 64 * NW - 1) / (64 * NW);
    static_assert(PIECES % 64 == 0, "whole waves copy");
    int off[JOBS];
    long long stride;         // bytes from row to row
    int row_bytes;
    __device__ __forceinline__ Copy(long long stride_elems, int d) {
        stride = stride_elems * (long long)sizeof(T);
        row_bytes = 2 * d * (int)sizeof(T);
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
        for (int j = 0; j < JOBS; ++j) {
            const int i = (j * NW + wave) * 64 + lane, row = i / L::NCH;
            const int piece = (i % L::NCH) ^ L::swz(row);
            const int half = piece / (L::NCH / 2), e = (piece % (L::NCH / 2)) * L::EPC;
            off[j] = e < d ? (int)(row * stride) + (half * d + e) * (int)sizeof(T) : (int)0x80000000;
        }
    }
    // rows row0 .. row0 + ROWS of `base`, of which those below `end` exist
    __device__ __forceinline__ void issue(const T* base, long long row0, long long end, char* dst) const {
        const long long have = end - row0 < ROWS ? end - row0 : ROWS;
        const unsigned bytes = have > 0 ? (unsigned)((have - 1) * stride) + (unsigned)row_bytes : 0u;
        const __amdgpu_buffer_rsrc_t rs =
            __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)base + row0 * stride), 0, bytes, 0x00020000);
        const int wave = threadIdx.x >> 6;
#pragma unroll
        for (int j = 0; j < JOBS; ++j)
            if (PIECES % (64 * NW) == 0 || (j * NW + wave) * 64 < PIECES)
                copy_piece(rs, dst + (j * NW + wave) * 1024, off[j]);
    }
};

// copies issued so far have landed in LDS, for every wave; nobody reads the buffer that is filled next
__device__ __forceinline__ void stage_sync() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// one operand row from global memory: columns [.., 8) of half `half`, zeros outside the head or for a missing row
template <typename T> __device__ __forceinline__ Frag<T> global_piece(const T* row, int half, int col, int d, bool have) {
    Frag<T> f;
    const bool ok = have && col < d;
    const T* p = row + (ok ? half * d + col : 0);
    if constexpr (sizeof(T) == 2) {
        bf16x8 z;
#pragma unroll
        for (int j = 0; j < 8; ++j) z[j] = (bf16)0.f;
        f.v = ok ? *reinterpret_cast<const bf16x8*>(p) : z;
    } else {
        const float4 z{0.f, 0.f, 0.f, 0.f};
        const float4 lo = ok ? *reinterpret_cast<const float4*>(p) : z, hi = ok ? *reinterpret_cast<const float4*>(p + 4) : z;
        f.v[0] = lo.x; f.v[1] = lo.y; f.v[2] = lo.z; f.v[3] = lo.w;
        f.v[4] = hi.x; f.v[5] = hi.y; f.v[6] = hi.z; f.v[7] = hi.w;
    }
    return f;
}

struct Strides { long long b, t, h; };      // elements
template <typename T> struct Args {
    const T* q; const T* k; const T* v;
    Strides qs, ks, vs;
    const void* lam;
    const int* lengths;
    T* o; T* o2; float* lse;                // o2 [B,Tq,H,2d] = O_2, lse f32 [B,H,Tq,2] (base 2): kept for the backward pass
    float* part;                            // partial results of a split key axis
    const T* dout; const T* o_in; const T* o2_in; const float* lse_in;
    float4* stat;                           // [B,H,Tq]: lse_1, lse_2, delta_1, delta_2
    T* dq; T* dk; T* dv;
    int lam_bf16, B, Tq, Tk, H, Hk, d, causal, nsplit;
    float scale, c;                         // c = scale * log2(e)
};

__device__ __forceinline__ float lam_of(const void* lam, int is_bf16, int h) {
    return is_bf16 ? (float)((const bf16*)lam)[h] : ((const float*)lam)[h];
}
template <typename T> __device__ __forceinline__ int keys_of(const Args<T>& a, int b) {
    if (!a.lengths) return a.Tk;
    const int n = a.lengths[b];
    return n < 0 ? 0 : n > a.Tk ? a.Tk : n;
}

// Workgroup id -> (batch and key/value head, tile).  Ids go round the 8 XCDs; when the heads divide by 8, all the tiles
// of a head stay on one XCD, whose L2 then holds that head's keys and values.
__device__ __forceinline__ void locate(int id, int heads, int tiles, int& bh, int& x) {
    if (heads % 8 == 0) {
        const int s = id >> 3;
        bh = (s / tiles) * 8 + (id & 7);
        x = s % tiles;
    } else {
        bh = id / tiles;
        x = id % tiles;
    }
}

__device__ __forceinline__ int wave_min_i(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
    return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_max_i(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o, 64));
    return __builtin_amdgcn_readfirstlane(v);
}

// stores 4 consecutive padded columns (c a multiple of 4) of a [2, d] row
template <typename T, int DP> __device__ __forceinline__ void store_cols(T* row, int c, int d, float x0, float x1, float x2, float x3) {
    const int half = c / DP, j = c % DP;
    if (j >= d) return;
    Vec4<T> v;
    v.set(0, x0); v.set(1, x1); v.set(2, x2); v.set(3, x3);
    v.store(row + half * d + j);
}

// ------------------------------------------------------------------------------ forward
// The query rows of all the heads that share a key/value head are one list, row r = token r / group, head r % group:
// one copy of the keys serves the whole group.  KEYS_SPLIT false: wave w takes rows 32 w .. of the workgroup's 128 and
// all keys of the tile.  KEYS_SPLIT true (at most 32 rows, single tokens): all waves take the same 32 rows and wave w
// the keys 32 w .. of the tile; the waves' results are joined through LDS at the end.
template <typename T, int DP, int NW, bool KEYS_SPLIT, int KT>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 2 ? 2 : 1) void attn_fwd_kernel(Args<T> a) {
    using L = Tile<T, DP>;
    constexpr int KS = DP / 16, DT = 2 * DP / 32;
    constexpr int RB = KEYS_SPLIT ? 32 : 32 * NW;
    constexpr int TB = KT * L::ROWB;                       // bytes of a key or value tile
    extern __shared__ __align__(16) char smem[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h2 = lane >> 5;
    const int group = a.H / a.Hk;
    const long long rows = (long long)group * a.Tq;
    const int tiles = (int)((rows + RB - 1) / RB) * a.nsplit;
    int bh, x;
    locate(blockIdx.x, a.B * a.Hk, tiles, bh, x);
    const int split = x % a.nsplit;
    const int rt = tiles / a.nsplit - 1 - x / a.nsplit;    // causal rows see more keys the later they are: longest first
    const int b = bh / a.Hk, hk = bh % a.Hk;
    const long long r0 = (long long)rt * RB;
    const long long row = r0 + (KEYS_SPLIT ? 0 : wave * 32) + (lane & 31);
    const bool have = row < rows;
    const long long rr = have ? row : rows - 1;            // lanes behind the last row repeat it
    const int t = (int)(rr / group), hq = hk * group + (int)(rr % group);
    const int kend = keys_of(a, b), reach = a.Tk - a.Tq;
    const int vis = a.causal ? max(0, min(kend, t + reach + 1)) : kend;     // the row sees keys [0, vis)
    const int vmin = wave_min_i(vis), vmax = wave_max_i(vis);
    const int t_last = (int)((r0 + RB < rows ? r0 + RB - 1 : rows - 1) / group);
    const int kstop = a.causal ? max(0, min(kend, t_last + reach + 1)) : kend;
    const int all = (kstop + KT - 1) / KT, per = (all + a.nsplit - 1) / a.nsplit;
    const int first = split * per, last = min(all, first + per);

    Frag<T> qf[2][KS];
    const T* qrow = a.q + b * a.qs.b + t * a.qs.t + hq * a.qs.h;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[i][s] = global_piece<T>(qrow, i, s * 16 + 8 * h2, a.d, true);

    f32x16 acc[2][DT];
    float m[2], l[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        m[i] = -1e30f;
        l[i] = 0.f;
#pragma unroll
        for (int n = 0; n < DT; ++n) acc[i][n] = zero16();
    }
    const T* const kbase = a.k + b * a.ks.b + hk * a.ks.h;
    const T* const vbase = a.v + b * a.vs.b + hk * a.vs.h;
    const Copy<T, DP, KT, NW> kc(a.ks.t, a.d), vc(a.vs.t, a.d);
    char* const buf0 = smem;
    char* const buf1 = smem + 2 * TB;

    auto sub_tile = [&](const char* kt, const char* vt, int sub, int key0) {
        if (key0 >= vmax) return;
        f32x16 s[2] = {zero16(), zero16()};
#pragma unroll
        for (int n = 0; n < KS; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                s[i] = mma(L::row_piece(kt, sub + (lane & 31), i * DP + n * 16 + 8 * h2), qf[i][n], s[i]);
        if (key0 + 32 > vmin) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const bool see = key0 + acc_row(r, h2) < vis;
                s[0][r] = see ? s[0][r] : -INFINITY;
                s[1][r] = see ? s[1][r] : -INFINITY;
            }
        }
        Frag<T> pf[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float top = s[i][0];
#pragma unroll
            for (int r = 1; r < 16; ++r) top = fmaxf(top, s[i][r]);
            top = fmaxf(top, __shfl_xor(top, 32, 64)) * a.c;
            // The maximum only has to keep the exponentials in range: it follows when a row outgrows it by 2^8, so the
            // accumulators are rescaled a few times per row instead of at every tile.
            if (__any(top > m[i] + 8.f)) {
                const float mn = fmaxf(m[i], top);
                const float f = exp2f(m[i] - mn);
                m[i] = mn;
                l[i] *= f;
#pragma unroll
                for (int n = 0; n < DT; ++n)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[i][n][r] *= f;
            }
            float p[16], sum = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                p[r] = __builtin_amdgcn_exp2f(s[i][r] * a.c - m[i]);
                sum += p[r];
            }
            l[i] += sum;
            pack(pf[i][0], p);
            pack(pf[i][1], p + 8);
        }
#pragma unroll
        for (int n = 0; n < DT; ++n)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const Frag<T> vf = L::col_piece(vt, sub + 16 * u, 32 * n, lane);
                acc[0][n] = mma(vf, pf[0][u], acc[0][n]);
                acc[1][n] = mma(vf, pf[1][u], acc[1][n]);
            }
    };
    // `cur` holds tile i, `fill` takes tile i + 1 (restrict: the reads need not wait for that copy)
    auto step = [&](int i, const char* __restrict__ cur, char* __restrict__ fill) {
        if (i + 1 < last) {
            kc.issue(kbase, (long long)(i + 1) * KT, kend, fill);
            vc.issue(vbase, (long long)(i + 1) * KT, kend, fill + TB);
        }
        if constexpr (KEYS_SPLIT) {
            sub_tile(cur, cur + TB, wave * 32, i * KT + wave * 32);
        } else {
#pragma unroll
            for (int u = 0; u < KT / 32; ++u) sub_tile(cur, cur + TB, u * 32, i * KT + u * 32);
        }
    };
    if (first < last) {
        kc.issue(kbase, (long long)first * KT, kend, buf0);
        vc.issue(vbase, (long long)first * KT, kend, buf0 + TB);
        for (int i = first;;) {
            stage_sync();
            step(i, buf0, buf1);
            if (++i >= last) break;
            stage_sync();
            step(i, buf1, buf0);
            if (++i >= last) break;
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) l[i] += __shfl_xor(l[i], 32, 64);

    if constexpr (KEYS_SPLIT) {
        // the waves' states one after the other into LDS, wave 0 adds them up
        float* const box = reinterpret_cast<float*>(smem);             // [2 DT 16][64] accumulators, then m, l
#pragma unroll 1
        for (int w = 1; w < NW; ++w) {
            __syncthreads();
            if (wave == w) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
#pragma unroll
                    for (int n = 0; n < DT; ++n)
#pragma unroll
                        for (int r = 0; r < 16; ++r) box[((i * DT + n) * 16 + r) * 64 + lane] = acc[i][n][r];
                    box[(2 * DT * 16 + 2 * i) * 64 + lane] = m[i];
                    box[(2 * DT * 16 + 2 * i + 1) * 64 + lane] = l[i];
                }
            }
            __syncthreads();
            if (wave == 0) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float mo = box[(2 * DT * 16 + 2 * i) * 64 + lane], lo = box[(2 * DT * 16 + 2 * i + 1) * 64 + lane];
                    const float mn = fmaxf(m[i], mo), f = exp2f(m[i] - mn), g = exp2f(mo - mn);
                    m[i] = mn;
                    l[i] = l[i] * f + lo * g;
#pragma unroll
                    for (int n = 0; n < DT; ++n)
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            acc[i][n][r] = acc[i][n][r] * f + box[((i * DT + n) * 16 + r) * 64 + lane] * g;
                }
            }
        }
        if (wave != 0) return;
    }
    if (!have) return;
    if (a.nsplit > 1) {
        const long long at = ((long long)bh * a.nsplit + split) * rows + row;
        float* const po = a.part + at * (4 * DP);
        float* const pm = a.part + (long long)a.B * a.Hk * a.nsplit * rows * (4 * DP) + at * 4;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int n = 0; n < DT; ++n)
#pragma unroll
                for (int r = 0; r < 16; r += 4)
                    *reinterpret_cast<float4*>(po + i * 2 * DP + 32 * n + acc_row(r, h2)) =
                        float4{acc[i][n][r], acc[i][n][r + 1], acc[i][n][r + 2], acc[i][n][r + 3]};
        if (h2 == 0) *reinterpret_cast<float4*>(pm) = float4{m[0], l[0], m[1], l[1]};
        return;
    }
    // a row that sees no key has l = 0: its output is zero, and its lse infinite, which makes its probabilities zero
    const float i1 = l[0] > 0.f || l[0] != l[0] ? 1.f / l[0] : 0.f, i2 = l[1] > 0.f || l[1] != l[1] ? 1.f / l[1] : 0.f;
    const float lam = lam_of(a.lam, a.lam_bf16, hq);
    const long long out = (((long long)b * a.Tq + t) * a.H + hq) * (2 * a.d);
#pragma unroll
    for (int n = 0; n < DT; ++n)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            float y[4], z[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                z[e] = acc[1][n][r + e] * i2;
                y[e] = acc[0][n][r + e] * i1 - lam * z[e];
            }
            store_cols<T, DP>(a.o + out, 32 * n + acc_row(r, h2), a.d, y[0], y[1], y[2], y[3]);
            if (a.o2) store_cols<T, DP>(a.o2 + out, 32 * n + acc_row(r, h2), a.d, z[0], z[1], z[2], z[3]);
        }
    if (a.lse && h2 == 0) {
        float* const p = a.lse + (((long long)b * a.H + hq) * a.Tq + t) * 2;
        p[0] = l[0] > 0.f ? m[0] + __log2f(l[0]) : l[0] == 0.f ? INFINITY : l[0];
        p[1] = l[1] > 0.f ? m[1] + __log2f(l[1]) : l[1] == 0.f ? INFINITY : l[1];
    }
}

// joins the partial results of a split key axis: one wave per query row
template <typename T, int DP> __global__ __launch_bounds__(256) void attn_join_kernel(Args<T> a) {
    const int lane = threadIdx.x & 63;
    const int group = a.H / a.Hk;
    const long long rows = (long long)group * a.Tq, id = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (id >= rows * a.B * a.Hk) return;
    const long long bh = id / rows, row = id % rows;
    const int b = (int)(bh / a.Hk), t = (int)(row / group), hq = (int)(bh % a.Hk) * group + (int)(row % group);
    const float* const pm = a.part + (long long)a.B * a.Hk * a.nsplit * rows * (4 * DP);
    float m[2] = {-1e30f, -1e30f};
    for (int s = 0; s < a.nsplit; ++s) {
        const float4 v = *reinterpret_cast<const float4*>(pm + ((bh * a.nsplit + s) * rows + row) * 4);
        m[0] = fmaxf(m[0], v.x);
        m[1] = fmaxf(m[1], v.z);
    }
    constexpr int NCOL = (2 * DP + 63) / 64;
    float l[2] = {0.f, 0.f}, acc[2][NCOL];
#pragma unroll
    for (int n = 0; n < NCOL; ++n) acc[0][n] = acc[1][n] = 0.f;
    for (int s = 0; s < a.nsplit; ++s) {
        const long long at = (bh * a.nsplit + s) * rows + row;
        const float4 v = *reinterpret_cast<const float4*>(pm + at * 4);
        const float f[2] = {exp2f(v.x - m[0]), exp2f(v.z - m[1])};
        l[0] += v.y * f[0];
        l[1] += v.w * f[1];
#pragma unroll
        for (int n = 0; n < NCOL; ++n) {
            const int c = n * 64 + lane;
            if (c < 2 * DP) {
                acc[0][n] += a.part[at * (4 * DP) + c] * f[0];
                acc[1][n] += a.part[at * (4 * DP) + 2 * DP + c] * f[1];
            }
        }
    }
    const float i1 = l[0] > 0.f || l[0] != l[0] ? 1.f / l[0] : 0.f, i2 = l[1] > 0.f || l[1] != l[1] ? 1.f / l[1] : 0.f;
    const float lam = lam_of(a.lam, a.lam_bf16, hq);
    const long long out = (((long long)b * a.Tq + t) * a.H + hq) * (2 * a.d);
#pragma unroll
    for (int n = 0; n < NCOL; ++n) {
        const int c = n * 64 + lane, half = c / DP, j = c % DP;
        if (c >= 2 * DP || j >= a.d) continue;
        const float z = acc[1][n] * i2, y = acc[0][n] * i1 - lam * z;
        a.o[out + half * a.d + j] = from_f32<T>(y);
        if (a.o2) a.o2[out + half * a.d + j] = from_f32<T>(z);
    }
    if (a.lse && lane < 2) {
        const float ll = lane ? l[1] : l[0], mm = lane ? m[1] : m[0];
        a.lse[(((long long)b * a.H + hq) * a.Tq + t) * 2 + lane] = ll > 0.f ? mm + __log2f(ll) : ll == 0.f ? INFINITY : ll;
    }
}

// ------------------------------------------------------------------------------ backward
// stat = (lse_1, lse_2, delta_1, delta_2) per row: delta_2 = do . O_2, delta_1 = do . o + lam delta_2.  16 lanes per row.
template <typename T> __global__ __launch_bounds__(256) void attn_delta_kernel(Args<T> a) {
    const long long id = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);       // row (b, t, h)
    const long long n = (long long)a.B * a.Tq * a.H;
    const int q = threadIdx.x & 15;
    const long long at = (id < n ? id : n - 1) * (2 * a.d) + 8 * q;
    float d1 = 0.f, d2 = 0.f;
    if (8 * q < 2 * a.d) {
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
            Vec4<T> g, o, o2;
            g.load(a.dout + at + j);
            o.load(a.o_in + at + j);
            o2.load(a.o2_in + at + j);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                d1 += g.get(e) * o.get(e);
                d2 += g.get(e) * o2.get(e);
            }
        }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
        d1 += __shfl_xor(d1, o, 64);
        d2 += __shfl_xor(d2, o, 64);
    }
    if (q != 0 || id >= n) return;
    const int h = (int)(id % a.H), t = (int)(id / a.H % a.Tq);
    const long long b = id / a.H / a.Tq, at_s = (b * a.H + h) * a.Tq + t;
    const float2 ls = *reinterpret_cast<const float2*>(a.lse_in + at_s * 2);
    a.stat[at_s] = float4{ls.x, ls.y, d1 + lam_of(a.lam, a.lam_bf16, h) * d2, d2};
}

// dlam[h] = -sum over the rows of head h of delta_2, in 64 bits and a fixed order
__global__ __launch_bounds__(256) void attn_dlam_kernel(const float4* __restrict__ stat, void* __restrict__ dlam, int lam_bf16,
                                                        int B, int H, int Tq) {
    __shared__ double sm[4];
    const int h = blockIdx.x;
    double s = 0.0;
    const long long n = (long long)B * Tq;
    for (long long i = threadIdx.x; i < n; i += 256) s += (double)stat[(i / Tq * H + h) * Tq + i % Tq].w;
    s = block_sum_256_d(s, sm);
    if (threadIdx.x == 0) {
        if (lam_bf16) ((bf16*)dlam)[h] = (bf16)(float)-s;
        else ((float*)dlam)[h] = (float)-s;
    }
}

// Gradient of the queries: as the forward pass, 32 rows per wave, the keys tile by tile.
template <typename T, int DP, int KT>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void attn_dq_kernel(Args<T> a) {
    using L = Tile<T, DP>;
    constexpr int NW = 4, RB = 32 * NW, KS = DP / 16, VS = 2 * DP / 16;
    constexpr int NA = DP == 16 ? 2 : 2 * DP / 32;         // accumulators: 32 columns each (DP = 16: both halves in each)
    constexpr int TB = KT * L::ROWB;
    extern __shared__ __align__(16) char smem[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h2 = lane >> 5;
    const int group = a.H / a.Hk;
    const long long rows = (long long)group * a.Tq;
    const int tiles = (int)((rows + RB - 1) / RB);
    int bh, x;
    locate(blockIdx.x, a.B * a.Hk, tiles, bh, x);
    const int rt = tiles - 1 - x;
    const int b = bh / a.Hk, hk = bh % a.Hk;
    const long long r0 = (long long)rt * RB, row = r0 + wave * 32 + (lane & 31);
    const bool have = row < rows;
    const long long rr = have ? row : rows - 1;
    const int t = (int)(rr / group), hq = hk * group + (int)(rr % group);
    const int kend = keys_of(a, b), reach = a.Tk - a.Tq;
    const int vis = a.causal ? max(0, min(kend, t + reach + 1)) : kend;
    const int vmin = wave_min_i(vis), vmax = wave_max_i(vis);
    const int t_last = (int)((r0 + RB < rows ? r0 + RB - 1 : rows - 1) / group);
    const int kstop = a.causal ? max(0, min(kend, t_last + reach + 1)) : kend;
    const int last = (kstop + KT - 1) / KT;

    Frag<T> qf[2][KS], gf[VS];
    const T* qrow = a.q + b * a.qs.b + t * a.qs.t + hq * a.qs.h;
    const long long out = (((long long)b * a.Tq + t) * a.H + hq) * (2 * a.d);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        qf[0][s] = global_piece<T>(qrow, 0, s * 16 + 8 * h2, a.d, true);
        qf[1][s] = global_piece<T>(qrow, 1, s * 16 + 8 * h2, a.d, true);
        gf[s] = global_piece<T>(a.dout + out, 0, s * 16 + 8 * h2, a.d, true);
        gf[KS + s] = global_piece<T>(a.dout + out, 1, s * 16 + 8 * h2, a.d, true);
    }
    const float4 st = a.stat[((long long)b * a.H + hq) * a.Tq + t];
    f32x16 acc[NA];
#pragma unroll
    for (int n = 0; n < NA; ++n) acc[n] = zero16();
    const T* const kbase = a.k + b * a.ks.b + hk * a.ks.h;
    const T* const vbase = a.v + b * a.vs.b + hk * a.vs.h;
    const Copy<T, DP, KT, NW> kc(a.ks.t, a.d), vc(a.vs.t, a.d);
    char* const buf0 = smem;
    char* const buf1 = smem + 2 * TB;

    auto sub_tile = [&](const char* kt, const char* vt, int sub, int key0) {
        if (key0 >= vmax) return;
        f32x16 s[2] = {zero16(), zero16()}, dp = zero16();
#pragma unroll
        for (int n = 0; n < KS; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                s[i] = mma(L::row_piece(kt, sub + (lane & 31), i * DP + n * 16 + 8 * h2), qf[i][n], s[i]);
#pragma unroll
        for (int n = 0; n < VS; ++n) dp = mma(L::row_piece(vt, sub + (lane & 31), n * 16 + 8 * h2), gf[n], dp);
        if (key0 + 32 > vmin) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const bool see = key0 + acc_row(r, h2) < vis;
                s[0][r] = see ? s[0][r] : -INFINITY;
                s[1][r] = see ? s[1][r] : -INFINITY;
            }
        }
        Frag<T> df[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float lse = i ? st.y : st.x, delta = i ? st.w : st.z;
            float ds[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) ds[r] = __builtin_amdgcn_exp2f(s[i][r] * a.c - lse) * (dp[r] - delta);
            pack(df[i][0], ds);
            pack(df[i][1], ds + 8);
        }
#pragma unroll
        for (int n = 0; n < NA; ++n)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int col = DP == 16 ? 0 : 32 * n, map = DP == 16 ? n : 32 * n / DP;
                acc[n] = mma(L::col_piece(kt, sub + 16 * u, col, lane), df[map][u], acc[n]);
            }
    };
    auto step = [&](int i, const char* __restrict__ cur, char* __restrict__ fill) {
        if (i + 1 < last) {
            kc.issue(kbase, (long long)(i + 1) * KT, kend, fill);
            vc.issue(vbase, (long long)(i + 1) * KT, kend, fill + TB);
        }
#pragma unroll
        for (int u = 0; u < KT / 32; ++u) sub_tile(cur, cur + TB, u * 32, i * KT + u * 32);
    };
    if (last > 0) {
        kc.issue(kbase, 0, kend, buf0);
        vc.issue(vbase, 0, kend, buf0 + TB);
        for (int i = 0;;) {
            stage_sync();
            step(i, buf0, buf1);
            if (++i >= last) break;
            stage_sync();
            step(i, buf1, buf0);
            if (++i >= last) break;
        }
    }
    if (!have) return;
    const float f1 = a.scale, f2 = -a.scale * lam_of(a.lam, a.lam_bf16, hq);
#pragma unroll
    for (int n = 0; n < NA; ++n)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int col = (DP == 16 ? 0 : 32 * n) + acc_row(r, h2), map = DP == 16 ? n : 32 * n / DP;
            const float f = map ? f2 : f1;
            if (col / DP == map)
                store_cols<T, DP>(a.dq + out, col, a.d, acc[n][r] * f, acc[n][r + 1] * f, acc[n][r + 2] * f, acc[n][r + 3] * f);
        }
}

// Gradients of the keys and values: a wave owns 32 keys (keys in registers, values in LDS), the workgroup's 128 keys
// meet the query rows of every head of the group 32 at a time.
template <typename T, int DP>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void attn_dkv_kernel(Args<T> a) {
    using L = Tile<T, DP>;
    constexpr int NW = 4, KB = 32 * NW, QT = 32, KS = DP / 16, VS = 2 * DP / 16, DT = 2 * DP / 32;
    constexpr int NA = DP == 16 ? 2 : DT;
    constexpr int TB = QT * L::ROWB, SB = 1024;            // query / gradient tile; row statistics (32 x 16 bytes, copied by a wave)
    constexpr int BUF = 2 * TB + SB;
    extern __shared__ __align__(16) char smem[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h2 = lane >> 5;
    const int group = a.H / a.Hk;
    const int tiles = (a.Tk + KB - 1) / KB;
    int bh, x;
    locate(blockIdx.x, a.B * a.Hk, tiles, bh, x);
    const int b = bh / a.Hk, hk = bh % a.Hk, k0 = x * KB;
    const int key = k0 + wave * 32 + (lane & 31);
    const int kend = keys_of(a, b), reach = a.Tk - a.Tq;
    const int t_min = a.causal ? max(0, key - reach) : 0;                  // the key is seen by queries [t_min, Tq)
    const int w_first = k0 + wave * 32;                                    // the wave's first key
    const int w_tmax = a.causal ? w_first + 31 - reach : 0;                // queries from here on see all keys of the wave
    const int q_first = a.causal ? max(0, k0 - reach) / QT : 0;            // first query tile that sees a key of the workgroup
    const int q_tiles = (a.Tq + QT - 1) / QT;
    const int per_head = k0 < kend && q_first < q_tiles ? q_tiles - q_first : 0;
    const int last = per_head * group;

    char* const vmem = smem;                                               // [KB] value rows
    char* const buf0 = smem + KB * L::ROWB;
    char* const buf1 = buf0 + BUF;
    const T* const kbase = a.k + b * a.ks.b + hk * a.ks.h;
    const T* const vbase = a.v + b * a.vs.b + hk * a.vs.h;
    Frag<T> kf[2][KS];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int s = 0; s < KS; ++s)
            kf[i][s] = global_piece<T>(kbase + (key < kend ? (long long)key * a.ks.t : 0), i, s * 16 + 8 * h2, a.d, key < kend);
    f32x16 dv[DT], dk[NA];
#pragma unroll
    for (int n = 0; n < DT; ++n) dv[n] = zero16();
#pragma unroll
    for (int n = 0; n < NA; ++n) dk[n] = zero16();

    const Copy<T, DP, QT, NW> qc(a.qs.t, a.d), gc((long long)a.H * 2 * a.d, a.d);
    const long long gstride = (long long)a.H * 2 * a.d;
    auto issue = [&](int i, char* dst) {
        const int hq = hk * group + i / per_head, qt = q_first + i % per_head;
        qc.issue(a.q + b * a.qs.b + hq * a.qs.h, (long long)qt * QT, a.Tq, dst);
        gc.issue(a.dout + (long long)b * a.Tq * gstride + hq * (2 * a.d), (long long)qt * QT, a.Tq, dst + TB);
        if (wave == 0) {
            const int left = a.Tq - qt * QT, n = left < QT ? left : QT;
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
                (void*)(a.stat + ((long long)b * a.H + hq) * a.Tq + qt * QT), 0, (unsigned)n * 16u, 0x00020000);
            copy_piece(rs, dst + 2 * TB, lane * 16);
        }
    };
    auto step = [&](int i, const char* __restrict__ cur, char* __restrict__ fill, const char* __restrict__ vals) {
        if (i + 1 < last) issue(i + 1, fill);
        const int t0 = (q_first + i % per_head) * QT;
        if (w_first >= kend || (a.causal && t0 + QT - 1 + reach < w_first)) return;     // nothing of this wave is seen
        const float lam = lam_of(a.lam, a.lam_bf16, hk * group + i / per_head);
        const char* const qt = cur;
        const char* const gt = cur + TB;
        const float4* const stat = reinterpret_cast<const float4*>(cur + 2 * TB);
        f32x16 s[2] = {zero16(), zero16()}, dp = zero16();
#pragma unroll
        for (int n = 0; n < KS; ++n)
#pragma unroll
            for (int u = 0; u < 2; ++u)
                s[u] = mma(L::row_piece(qt, lane & 31, u * DP + n * 16 + 8 * h2), kf[u][n], s[u]);
#pragma unroll
        for (int n = 0; n < VS; ++n)
            dp = mma(L::row_piece(gt, lane & 31, n * 16 + 8 * h2), L::row_piece(vals, wave * 32 + (lane & 31), n * 16 + 8 * h2), dp);
        const bool edge = w_first + 32 > kend || (a.causal && t0 < w_tmax);
        if (edge) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const bool see = key < kend && t0 + acc_row(r, h2) >= t_min;
                s[0][r] = see ? s[0][r] : -INFINITY;
                s[1][r] = see ? s[1][r] : -INFINITY;
            }
        }
        Frag<T> pf[2], df[2][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float p[8], d1[8], d2[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int r = 8 * u + j;
                const float4 st = stat[acc_row(r, h2)];
                const float p1 = __builtin_amdgcn_exp2f(s[0][r] * a.c - st.x);
                const float p2 = -lam * __builtin_amdgcn_exp2f(s[1][r] * a.c - st.y);
                p[j] = p1 + p2;
                d1[j] = p1 * (dp[r] - st.z);
                d2[j] = p2 * (dp[r] - st.w);
            }
            pack(pf[u], p);
            pack(df[0][u], d1);
            pack(df[1][u], d2);
        }
#pragma unroll
        for (int n = 0; n < DT; ++n)
#pragma unroll
            for (int u = 0; u < 2; ++u) dv[n] = mma(L::col_piece(gt, 16 * u, 32 * n, lane), pf[u], dv[n]);
#pragma unroll
        for (int n = 0; n < NA; ++n)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int col = DP == 16 ? 0 : 32 * n, map = DP == 16 ? n : 32 * n / DP;
                dk[n] = mma(L::col_piece(qt, 16 * u, col, lane), df[map][u], dk[n]);
            }
    };
    if (last > 0) {
        const Copy<T, DP, KB, NW> vc(a.vs.t, a.d);
        vc.issue(vbase, k0, kend, vmem);
        issue(0, buf0);
        for (int i = 0;;) {
            stage_sync();
            step(i, buf0, buf1, vmem);
            if (++i >= last) break;
            stage_sync();
            step(i, buf1, buf0, vmem);
            if (++i >= last) break;
        }
    }
    if (key >= a.Tk) return;
    const long long out = (((long long)b * a.Tk + key) * a.Hk + hk) * (2 * a.d);
#pragma unroll
    for (int n = 0; n < DT; ++n)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
            store_cols<T, DP>(a.dv + out, 32 * n + acc_row(r, h2), a.d, dv[n][r], dv[n][r + 1], dv[n][r + 2], dv[n][r + 3]);
#pragma unroll
    for (int n = 0; n < NA; ++n)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int col = (DP == 16 ? 0 : 32 * n) + acc_row(r, h2), map = DP == 16 ? n : 32 * n / DP;
            if (col / DP == map)
                store_cols<T, DP>(a.dk + out, col, a.d, dk[n][r] * a.scale, dk[n][r + 1] * a.scale, dk[n][r + 2] * a.scale,
                                  dk[n][r + 3] * a.scale);
        }
}

// ------------------------------------------------------------------------------ host side
int padded(int d) { return d <= 16 ? 16 : d <= 32 ? 32 : 64; }

int check_desc(const sf_diff_attn_desc* p, const char* who) {
    SF_REQUIRE(p, "%s: null descriptor", who);
    SF_REQUIRE(p->dtype == SF_F32 || p->dtype == SF_BF16, "%s: unknown dtype %d", who, p->dtype);
    SF_REQUIRE(p->lam_dtype == SF_F32 || p->lam_dtype == SF_BF16, "%s: unknown dtype %d of lam", who, p->lam_dtype);
    SF_REQUIRE(p->d >= 8 && p->d <= 64 && p->d % 8 == 0, "%s: d = %d is not a multiple of 8 up to 64", who, p->d);
    SF_REQUIRE(p->B > 0 && p->Tq > 0 && p->Tk > 0 && p->H > 0 && p->Hk > 0 && p->H % p->Hk == 0,
               "%s: bad sizes (B %d, Tq %d, Tk %d, H %d, Hk %d)", who, p->B, p->Tq, p->Tk, p->H, p->Hk);
    SF_REQUIRE(p->Tq <= (1 << 24) && p->Tk <= (1 << 24) && p->H <= (1 << 16) && p->B <= (1 << 24),
               "%s: sizes beyond 2^24 tokens, 2^24 samples or 2^16 heads", who);
    SF_REQUIRE((long long)p->H * 2 * p->d < (1 << 22), "%s: H * 2 d = %lld is not below 2^22", who, (long long)p->H * 2 * p->d);
    SF_REQUIRE(p->scale > 0.f && p->scale < 1e30f, "%s: scale must be positive", who);
    const long long epc = p->dtype == SF_BF16 ? 8 : 4;
    for (int i = 0; i < 9; ++i) {
        const long long s = i < 3 ? p->q_stride[i] : i < 6 ? p->k_stride[i - 3] : p->v_stride[i - 6];
        SF_REQUIRE(s >= 0 && s % epc == 0, "%s: stride %lld is not a multiple of 16 bytes", who, s);
        SF_REQUIRE(i % 3 != 1 || (s >= 2 * p->d && s < (1 << 22)), "%s: token stride %lld (a head has %d values)", who, s, 2 * p->d);
    }
    const double groups = (double)p->B * p->Hk * (((double)p->H / p->Hk * p->Tq + 31) / 32 + (p->Tk + 127) / 128);
    SF_REQUIRE(groups < 1e8 && (double)p->B * p->Tq * p->H < 2e9, "%s: too many rows", who);
    return SF_OK;
}
int check_align(const void* const* ps, int n, const char* who) {
    for (int i = 0; i < n; ++i) SF_REQUIRE(ps[i] && (uintptr_t)ps[i] % 16 == 0, "%s: pointer %d is null or not 16-byte aligned", who, i);
    return SF_OK;
}

// How the forward pass is cut.  Up to 32 query rows per key/value head the waves share out the keys of a tile (one copy
// of the keys, four waves' worth of loads in flight per workgroup), beyond that the rows.  When the rows alone give
// fewer than two workgroups per CU the key axis is split so that they do, as long as a part keeps two tiles.
struct FwdPlan { bool keys; int kt, rb, nsplit; };
FwdPlan fwd_plan(const sf_diff_attn_desc* p) {
    const long long rows = (long long)(p->H / p->Hk) * p->Tq;
    const bool f32 = p->dtype == SF_F32;
    FwdPlan f;
    f.keys = rows <= 32;
    f.kt = f.keys ? (f32 && padded(p->d) == 64 ? 64 : 128) : f32 ? 32 : 64;
    f.rb = f.keys ? 32 : 128;
    const long long groups = (rows + f.rb - 1) / f.rb * p->B * p->Hk;
    const int key_tiles = (p->Tk + f.kt - 1) / f.kt;
    long long n = groups >= 512 ? 1 : (512 + groups - 1) / groups;
    if (n > key_tiles / 2) n = key_tiles / 2;
    if (n > 128) n = 128;
    f.nsplit = n < 1 ? 1 : (int)n;
    return f;
}

template <typename T> Args<T> make_args(const sf_diff_attn_desc* p, const void* q, const void* k, const void* v, const void* lam,
                                        const int* lengths) {
    Args<T> a{};
    a.q = (const T*)q; a.k = (const T*)k; a.v = (const T*)v;
    a.qs = {p->q_stride[0], p->q_stride[1], p->q_stride[2]};
    a.ks = {p->k_stride[0], p->k_stride[1], p->k_stride[2]};
    a.vs = {p->v_stride[0], p->v_stride[1], p->v_stride[2]};
    a.lam = lam; a.lam_bf16 = p->lam_dtype == SF_BF16; a.lengths = lengths;
    a.B = p->B; a.Tq = p->Tq; a.Tk = p->Tk; a.H = p->H; a.Hk = p->Hk; a.d = p->d; a.causal = p->causal != 0;
    a.nsplit = 1;
    a.scale = p->scale;
    a.c = (float)((double)p->scale * 1.4426950408889634);
    return a;
}

template <typename K> int allow_lds(K kernel, int bytes) {
    if (hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) {
        sf_set_error("sf_diff_attn: %d bytes of LDS refused", bytes);
        return SF_ELAUNCH;
    }
    return SF_OK;
}
#define SF_LDS_ONCE(kernel, bytes)                                    \
    do {                                                              \
        static DeviceOnce once;                                       \
        if (!once.done()) {                                           \
            if (int rc = allow_lds(kernel, bytes)) return rc;         \
            once.mark();                                              \
        }                                                             \
    } while (0)

template <typename T, int DP> int launch_fwd(Args<T> a, const FwdPlan& f, hipStream_t st) {
    const long long rows = (long long)(a.H / a.Hk) * a.Tq;
    const int grid = (int)((rows + f.rb - 1) / f.rb) * a.B * a.Hk * f.nsplit;
    constexpr int ROWB = Tile<T, DP>::ROWB;
    a.nsplit = f.nsplit;
    if (f.keys) {
        constexpr int NW = sizeof(T) == 4 && DP == 64 ? 2 : 4, KT = 32 * NW;
        constexpr int box = (2 * (2 * DP / 32) * 16 + 4) * 64 * 4;
        constexpr int lds = 4 * KT * ROWB > box ? 4 * KT * ROWB : box;
        SF_LDS_ONCE((attn_fwd_kernel<T, DP, NW, true, KT>), lds);
        hipLaunchKernelGGL((attn_fwd_kernel<T, DP, NW, true, KT>), dim3(grid), dim3(64 * NW), lds, st, a);
    } else {
        constexpr int KT = sizeof(T) == 4 ? 32 : 64, lds = 4 * KT * ROWB;
        SF_LDS_ONCE((attn_fwd_kernel<T, DP, 4, false, KT>), lds);
        hipLaunchKernelGGL((attn_fwd_kernel<T, DP, 4, false, KT>), dim3(grid), dim3(256), lds, st, a);
    }
    SF_LAUNCH_CHECK("sf_diff_attn_fwd");
    if (f.nsplit > 1) {
        hipLaunchKernelGGL((attn_join_kernel<T, DP>), dim3(ceil_div(rows * a.B * a.Hk, 4)), dim3(256), 0, st, a);
        SF_LAUNCH_CHECK("sf_diff_attn_fwd (join)");
    }
    return SF_OK;
}

template <typename T, int DP> int launch_bwd(const Args<T>& a, hipStream_t st) {
    const long long rows = (long long)(a.H / a.Hk) * a.Tq, n = (long long)a.B * a.Tq * a.H;
    constexpr int ROWB = Tile<T, DP>::ROWB, KT = sizeof(T) == 4 ? 32 : 64;
    hipLaunchKernelGGL((attn_delta_kernel<T>), dim3(ceil_div(n, 16)), dim3(256), 0, st, a);
    SF_LAUNCH_CHECK("sf_diff_attn_bwd (delta)");
    constexpr int lds_q = 4 * KT * ROWB, lds_k = 128 * ROWB + 2 * (2 * 32 * ROWB + 1024);
    SF_LDS_ONCE((attn_dq_kernel<T, DP, KT>), lds_q);
    hipLaunchKernelGGL((attn_dq_kernel<T, DP, KT>), dim3(ceil_div(rows, 128) * a.B * a.Hk), dim3(256), lds_q, st, a);
    SF_LAUNCH_CHECK("sf_diff_attn_bwd (queries)");
    SF_LDS_ONCE((attn_dkv_kernel<T, DP>), lds_k);
    hipLaunchKernelGGL((attn_dkv_kernel<T, DP>), dim3(ceil_div(a.Tk, 128) * a.B * a.Hk), dim3(256), lds_k, st, a);
    SF_LAUNCH_CHECK("sf_diff_attn_bwd (keys)");
    return SF_OK;
}

template <typename T> int fwd(const sf_diff_attn_desc* p, const void* q, const void* k, const void* v, const void* lam,
                              const int* lengths, void* o, void* o2, float* lse, float* part, hipStream_t st) {
    Args<T> a = make_args<T>(p, q, k, v, lam, lengths);
    a.o = (T*)o; a.o2 = (T*)o2; a.lse = lse; a.part = part;
    const FwdPlan f = fwd_plan(p);
    const int dp = padded(p->d);
    return dp == 16 ? launch_fwd<T, 16>(a, f, st) : dp == 32 ? launch_fwd<T, 32>(a, f, st) : launch_fwd<T, 64>(a, f, st);
}
template <typename T> int bwd(const sf_diff_attn_desc* p, const void* q, const void* k, const void* v, const void* lam,
                              const int* lengths, const void* o, const void* o2, const float* lse, const void* dout, void* dq,
                              void* dk, void* dv, void* dlam, float4* stat, hipStream_t st) {
    Args<T> a = make_args<T>(p, q, k, v, lam, lengths);
    a.o_in = (const T*)o; a.o2_in = (const T*)o2; a.lse_in = lse; a.dout = (const T*)dout; a.stat = stat;
    a.dq = (T*)dq; a.dk = (T*)dk; a.dv = (T*)dv;
    const int dp = padded(p->d);
    if (int rc = dp == 16 ? launch_bwd<T, 16>(a, st) : dp == 32 ? launch_bwd<T, 32>(a, st) : launch_bwd<T, 64>(a, st)) return rc;
    if (dlam) {
        hipLaunchKernelGGL(attn_dlam_kernel, dim3(a.H), dim3(256), 0, st, stat, dlam, a.lam_bf16, a.B, a.H, a.Tq);
        SF_LAUNCH_CHECK("sf_diff_attn_bwd (lam)");
    }
    return SF_OK;
}

}  // namespace

extern "C" size_t sf_diff_attn_fwd_workspace_bytes(const sf_diff_attn_desc* p) {
    if (check_desc(p, "sf_diff_attn_fwd_workspace_bytes")) return 0;
    const FwdPlan f = fwd_plan(p);
    if (f.nsplit == 1) return 0;
    return (size_t)p->B * p->H * p->Tq * f.nsplit * (4 * padded(p->d) + 4) * sizeof(float);
}

extern "C" int sf_diff_attn_fwd(const sf_diff_attn_desc* p, const void* q, const void* k, const void* v, const void* lam,
                                const int* lengths, void* o, void* o2, float* lse, void* ws, size_t ws_bytes, void* stream) {
    if (int rc = check_desc(p, "sf_diff_attn_fwd")) return rc;
    const void* ps[] = {q, k, v, o};
    if (int rc = check_align(ps, 4, "sf_diff_attn_fwd")) return rc;
    SF_REQUIRE(lam && (!o2 == !lse) && (uintptr_t)o2 % 16 == 0, "sf_diff_attn_fwd: lam is missing, or o2 and lse are not both given");
    const size_t need = sf_diff_attn_fwd_workspace_bytes(p);
    SF_REQUIRE(!need || (ws && ws_bytes >= need && (uintptr_t)ws % 16 == 0), "sf_diff_attn_fwd: workspace of %zu bytes is too small (%zu)",
               ws_bytes, need);
    return p->dtype == SF_BF16 ? fwd<bf16>(p, q, k, v, lam, lengths, o, o2, lse, (float*)ws, (hipStream_t)stream)
                               : fwd<float>(p, q, k, v, lam, lengths, o, o2, lse, (float*)ws, (hipStream_t)stream);
}

extern "C" size_t sf_diff_attn_bwd_workspace_bytes(const sf_diff_attn_desc* p) {
    if (check_desc(p, "sf_diff_attn_bwd_workspace_bytes")) return 0;
    return (size_t)p->B * p->H * p->Tq * sizeof(float4);
}

extern "C" int sf_diff_attn_bwd(const sf_diff_attn_desc* p, const void* q, const void* k, const void* v, const void* lam,
                                const int* lengths, const void* o, const void* o2, const float* lse, const void* dout, void* dq,
                                void* dk, void* dv, void* dlam, void* ws, size_t ws_bytes, void* stream) {
    if (int rc = check_desc(p, "sf_diff_attn_bwd")) return rc;
    const void* ps[] = {q, k, v, o, o2, dout, dq, dk, dv, lse};
    if (int rc = check_align(ps, 10, "sf_diff_attn_bwd")) return rc;
    const size_t need = sf_diff_attn_bwd_workspace_bytes(p);
    SF_REQUIRE(lam && ws && ws_bytes >= need && (uintptr_t)ws % 16 == 0, "sf_diff_attn_bwd: workspace of %zu bytes is too small (%zu)",
               ws_bytes, need);
    return p->dtype == SF_BF16
               ? bwd<bf16>(p, q, k, v, lam, lengths, o, o2, lse, dout, dq, dk, dv, dlam, (float4*)ws, (hipStream_t)stream)
               : bwd<float>(p, q, k, v, lam, lengths, o, o2, lse, dout, dq, dk, dv, dlam, (float4*)ws, (hipStream_t)stream);
}
