// LayerNorm over the last axis, forward and backward, for any row count and width, f32 or bf16 rows with
// f32 weights, with the residual add in front of it fused in:
//
//   s = round(x + residual)   (round: to the rows' type, because that is what the next layer reads)
//   mu = mean(s),  var = mean((s - mu)^2),  r = 1 / sqrt(var + eps),  xh = (s - mu) r,  y = w xh + b
//   backward, g = w dy:  ds_total = r (g - mean(g) - xh mean(g xh)) + ds,  dw = sum_rows dy xh,  db = sum_rows dy
//
// All statistics and sums are f32; values are rounded to bf16 once, at the store.  A row's first mean is off by a few f32 steps of
// its size, which for rows far from zero may be more than their spread (0.05 at 1e5, where sqrt(eps) is 0.003): the centred
// values' own mean, summed beside their squares, takes that out of the values, the variance and the mean that is kept.
// Both directions are bound by HBM: rows of up to 8192 values are read and every array written exactly once,
// because a row lives in registers between its statistics and its output.
// A row belongs to G lanes (8 to 64 lanes of a wave, or the 256 threads of a workgroup), each holding NC
// pieces of 16 bytes; G and NC follow from the width alone (row_plan).  Workgroups are persistent: a lane's
// columns never change, so the weights and, backward, the sums of dw and db stay in its registers over all
// its rows.  The workgroups' partial dw / db rows go to a workspace and are folded in a fixed order by a
// second launch: no atomics, the same result every time.
//
// Measured (a copy of 1 GiB runs at 5.05 TB/s on the same card):
//   163840 x 256 bf16, residual, no statistics kept: 58 us, 335 MB, 5.8 TB/s
//   16384 x 4096 bf16, residual: forward 106 us, 537 MB, 5.1 TB/s; backward 108 us, 537 MB, 5.0 TB/s, and 4 us for the fold
//   30011 x 999 f32: forward 41 us, 240 MB, 5.9 TB/s; backward 71 us, 360 MB, 5.0 TB/s, and 5 us for the fold
//   160 x 128 bf16: 4, 6 and 3 us, all of it launch and latency
#include "sf_common.h"
#include <float.h>
#include "../../include/sfhip.h"

namespace {

constexpr int NT = 256;
constexpr int MAX_PARTS = 1024;          // partial dw / db rows of one backward call at most

// V consecutive elements at an address aligned to one element only: the hardware serves 16-byte global
// accesses at any element alignment, so odd widths and offset views keep the wide loads.
template <typename T, int V> struct __attribute__((packed, aligned(sizeof(T)))) Raw { T e[V]; };

template <typename T, int V> __device__ __forceinline__ void load_vec(const T* __restrict__ p, float* o) {
    const Raw<T, V> r = *reinterpret_cast<const Raw<T, V>*>(p);
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = to_f32(r.e[j]);
}
template <typename T, int V> __device__ __forceinline__ void store_vec(T* __restrict__ p, const float* v) {
    Raw<T, V> r;
#pragma unroll
    for (int j = 0; j < V; ++j) r.e[j] = from_f32<T>(v[j]);
    *reinterpret_cast<Raw<T, V>*>(p) = r;
}

// sum over the G lanes of a row, the result in every one of them (sm: 4 floats, G = 256 only)
template <int G> __device__ __forceinline__ float row_sum(float v, float* sm) {
    if constexpr (G == NT) return block_sum_256(v, sm);
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// the same of two values at once (sm: 8 floats)
template <int G> __device__ __forceinline__ void row_sums(float& a, float& b, float* sm) {
#pragma unroll
    for (int o = (G < 64 ? G : 64) / 2; o > 0; o >>= 1) {
        a += __shfl_xor(a, o, 64);
        b += __shfl_xor(b, o, 64);
    }
    if constexpr (G == NT) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) {
            sm[threadIdx.x >> 6] = a;
            sm[4 + (threadIdx.x >> 6)] = b;
        }
        __syncthreads();
        a = sm[0] + sm[1] + sm[2] + sm[3];
        b = sm[4] + sm[5] + sm[6] + sm[7];
    }
}

// a row's statistic where whole waves share a row: a scalar register
template <int G> __device__ __forceinline__ float shared(float v) {
    if constexpr (G >= 64) return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v)));
    return v;
}

// Columns of piece c of lane q: V elements from `col`.  The last piece of a row whose width V does not
// divide is moved back to end with the row; its first `skip` elements belong to the piece before it and
// are left out of the sums (their outputs are written twice, with the same bits).  A lane without a piece
// works on piece 0 of the row with everything skipped.  FULL: G * NC * V is the width, nothing is ever skipped (without
// the selects, and with dsum loaded early, the backward pass of 16384 x 4096 bf16 went from 136 to 110 us).
template <int G, int NC, int V, bool FULL> struct Cols {
    int col[NC], skip[NC];
    bool live[NC];
    __device__ __forceinline__ Cols(int q, int D) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int at = (q + c * G) * V;
            if constexpr (FULL) {
                col[c] = at;
                skip[c] = 0;
                live[c] = true;
                continue;
            }
            live[c] = at < D;
            col[c] = live[c] ? (at + V <= D ? at : D - V) : 0;
            skip[c] = live[c] ? at - col[c] : V;
        }
    }
};

template <typename T, int G, int NC, int V, bool FULL>
__global__ __launch_bounds__(NT) void norm_fwd_kernel(const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ sum,
                                                      const float* __restrict__ w, const float* __restrict__ b,
                                                      T* __restrict__ y, float* __restrict__ mean_out,
                                                      float* __restrict__ rstd_out, long long rows, int D, float eps) {
    __shared__ float sm[8];
    constexpr int RPB = NT / G;
    const int q = threadIdx.x % G;
    const Cols<G, NC, V, FULL> C(q, D);
    float wv[NC][V], bv[NC][V];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        if (w) load_vec<float, V>(w + C.col[c], wv[c]);
        if (b) load_vec<float, V>(b + C.col[c], bv[c]);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (!w) wv[c][j] = 1.f;
            if (!b) bv[c][j] = 0.f;
        }
    }
    const float count = (float)D;       // (divided by: a rounded reciprocal would put the mean of equal values off them)
    for (long long r0 = (long long)blockIdx.x * RPB; r0 < rows; r0 += (long long)gridDim.x * RPB) {
        const long long row = r0 + threadIdx.x / G;
        const bool have = row < rows;                     // lanes behind the last row repeat it without a store
        const long long at = (have ? row : rows - 1) * D;
        float v[NC][V];
#pragma unroll
        for (int c = 0; c < NC; ++c) load_vec<T, V>(x + at + C.col[c], v[c]);
        if (res) {
            float t[NC][V];
#pragma unroll
            for (int c = 0; c < NC; ++c) load_vec<T, V>(res + at + C.col[c], t[c]);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
#pragma unroll
                for (int j = 0; j < V; ++j) v[c][j] = to_f32(from_f32<T>(v[c][j] + t[c][j]));
                if (have && C.live[c]) store_vec<T, V>(sum + at + C.col[c], v[c]);
            }
        }
        float a = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int j = 0; j < V; ++j) a += j >= C.skip[c] ? v[c][j] : 0.f;
        const float mean = shared<G>(row_sum<G>(a, sm) / count);
        a = 0.f;
        float off = 0.f;                                  // mean of the centred values
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[c][j] -= mean;
                a += j >= C.skip[c] ? v[c][j] * v[c][j] : 0.f;
                off += j >= C.skip[c] ? v[c][j] : 0.f;
            }
        row_sums<G>(a, off, sm);
        off = shared<G>(off / count);
        // (squares that overflow leave an infinite variance, not inf - inf)
        const float rstd = shared<G>(1.0f / sqrtf(fmaxf(a / count - fminf(off * off, FLT_MAX), 0.f) + eps));
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
            for (int j = 0; j < V; ++j) v[c][j] = (v[c][j] - off) * rstd * wv[c][j] + bv[c][j];
            if (have && C.live[c]) store_vec<T, V>(y + at + C.col[c], v[c]);
        }
        if (mean_out && have && q == 0) {
            mean_out[row] = mean + off;
            rstd_out[row] = rstd;
        }
    }
}

template <typename T, int G, int NC, int V, bool FULL>
__global__ __launch_bounds__(NT) void norm_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ dsum,
                                                      const T* __restrict__ s, const float* __restrict__ w,
                                                      const float* __restrict__ mean, const float* __restrict__ rstd,
                                                      T* __restrict__ dx, float* __restrict__ part, long long rows, int D) {
    constexpr int RPB = NT / G;
    __shared__ float sm[4];
    __shared__ float fold[G < NT ? 3 * 64 * NC * V : 1];
    const int q = threadIdx.x % G;
    const Cols<G, NC, V, FULL> C(q, D);
    float wv[NC][V], aw[NC][V], ab[NC][V];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        if (w) load_vec<float, V>(w + C.col[c], wv[c]);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (!w) wv[c][j] = 1.f;
            aw[c][j] = ab[c][j] = 0.f;
        }
    }
    const float inv = 1.0f / (float)D;
    for (long long r0 = (long long)blockIdx.x * RPB; r0 < rows; r0 += (long long)gridDim.x * RPB) {
        const long long row = r0 + threadIdx.x / G;
        const bool have = row < rows;
        const long long rr = have ? row : rows - 1, at = rr * D;
        const float mu = mean[rr], rs = rstd[rr];
        float h[NC][V], g[NC][V];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            load_vec<T, V>(s + at + C.col[c], h[c]);
            load_vec<T, V>(dy + at + C.col[c], g[c]);
        }
        Raw<T, V> t[NC];            // (asked for before the sums, so that it is there behind them)
        if (dsum) {
#pragma unroll
            for (int c = 0; c < NC; ++c) t[c] = *reinterpret_cast<const Raw<T, V>*>(dsum + at + C.col[c]);
        }
        float m1 = 0.f, m2 = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                h[c][j] = (h[c][j] - mu) * rs;
                if (have) {
                    aw[c][j] += g[c][j] * h[c][j];
                    ab[c][j] += g[c][j];
                }
                g[c][j] *= wv[c][j];
                m1 += j >= C.skip[c] ? g[c][j] : 0.f;
                m2 += j >= C.skip[c] ? g[c][j] * h[c][j] : 0.f;
            }
        m1 = row_sum<G>(m1, sm) * inv;
        m2 = row_sum<G>(m2, sm) * inv;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                g[c][j] = rs * (g[c][j] - m1 - h[c][j] * m2);
                if (dsum) g[c][j] += to_f32(t[c].e[j]);
            }
            if (have && C.live[c]) store_vec<T, V>(dx + at + C.col[c], g[c]);
        }
    }
    if (!part) return;
    // sums of the workgroup's row groups: lanes of one wave that hold the same columns, then the four waves
    float* const out = part + (size_t)blockIdx.x * 2 * D;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        float (&acc)[NC][V] = k == 0 ? aw : ab;
        if constexpr (G < NT) {
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int j = 0; j < V; ++j) {
#pragma unroll
                    for (int o = G; o < 64; o <<= 1) acc[c][j] += __shfl_xor(acc[c][j], o, 64);
                }
            const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
            __syncthreads();
            if (wave > 0 && lane < G) {
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int j = 0; j < V; ++j) fold[((wave - 1) * NC * V + c * V + j) * 64 + lane] = acc[c][j];
            }
            __syncthreads();
            if (wave == 0 && lane < G) {
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int j = 0; j < V; ++j) {
#pragma unroll
                        for (int u = 0; u < 3; ++u) acc[c][j] += fold[(u * NC * V + c * V + j) * 64 + lane];
                    }
            }
        }
        if (threadIdx.x < G) {
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (j >= C.skip[c]) out[(size_t)k * D + C.col[c] + j] = acc[c][j];
        }
    }
}

// Rows wider than the registers of a workgroup hold: one workgroup per row, the row read again for each of
// its passes (three forward, two backward; from the L2 as far as it reaches).  A thread adds up to 65536 values one after the
// other: in 64 bits.
template <typename T>
__global__ __launch_bounds__(NT) void norm_fwd_wide_kernel(const T* __restrict__ x, const T* __restrict__ res,
                                                           T* __restrict__ sum, const float* __restrict__ w,
                                                           const float* __restrict__ b, T* __restrict__ y,
                                                           float* __restrict__ mean_out, float* __restrict__ rstd_out,
                                                           long long rows, int D, float eps) {
    __shared__ double sm[4];
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* xr = x + row * D;
        const T* rr = res ? res + row * D : nullptr;
        auto value = [&](int i) { return rr ? to_f32(from_f32<T>(to_f32(xr[i]) + to_f32(rr[i]))) : to_f32(xr[i]); };
        double a = 0.0;
        for (int i = threadIdx.x; i < D; i += NT) a += (double)value(i);
        const float mean = (float)(block_sum_256_d(a, sm) / D);
        double q = 0.0;
        a = 0.0;
        for (int i = threadIdx.x; i < D; i += NT) {
            const double c = (double)(value(i) - mean);
            q += c * c;
            a += c;
        }
        a = block_sum_256_d(a, sm) / D;
        q = block_sum_256_d(q, sm) / D - a * a;
        const float off = (float)a, rstd = 1.0f / sqrtf((float)fmax(q, 0.0) + eps);
        for (int i = threadIdx.x; i < D; i += NT) {
            const float v = value(i);
            if (rr) sum[row * D + i] = from_f32<T>(v);
            y[row * D + i] = from_f32<T>((v - mean - off) * rstd * (w ? w[i] : 1.f) + (b ? b[i] : 0.f));
        }
        if (mean_out && threadIdx.x == 0) {
            mean_out[row] = mean + off;
            rstd_out[row] = rstd;
        }
    }
}
template <typename T>
__global__ __launch_bounds__(NT) void norm_bwd_wide_kernel(const T* __restrict__ dy, const T* __restrict__ dsum,
                                                           const T* __restrict__ s, const float* __restrict__ w,
                                                           const float* __restrict__ mean, const float* __restrict__ rstd,
                                                           T* __restrict__ dx, long long rows, int D) {
    __shared__ double sm[4];
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const float mu = mean[row], rs = rstd[row];
        double g1 = 0.0, g2 = 0.0;
        for (int i = threadIdx.x; i < D; i += NT) {
            const float g = to_f32(dy[row * D + i]) * (w ? w[i] : 1.f);
            g1 += (double)g;
            g2 += (double)(g * ((to_f32(s[row * D + i]) - mu) * rs));
        }
        const float m1 = (float)(block_sum_256_d(g1, sm) / D), m2 = (float)(block_sum_256_d(g2, sm) / D);
        for (int i = threadIdx.x; i < D; i += NT) {
            const float g = to_f32(dy[row * D + i]) * (w ? w[i] : 1.f);
            float v = rs * (g - m1 - (to_f32(s[row * D + i]) - mu) * rs * m2);
            if (dsum) v += to_f32(dsum[row * D + i]);
            dx[row * D + i] = from_f32<T>(v);
        }
    }
}
// partial dw / db of rows [blockIdx.y * per, + per) for 256 columns (the wide rows' companion)
template <typename T>
__global__ __launch_bounds__(NT) void norm_bwd_cols_kernel(const T* __restrict__ dy, const T* __restrict__ s,
                                                           const float* __restrict__ mean, const float* __restrict__ rstd,
                                                           float* __restrict__ part, long long rows, long long per, int D) {
    const int c = blockIdx.x * NT + threadIdx.x;
    if (c >= D) return;
    const long long r0 = blockIdx.y * per, r1 = r0 + per < rows ? r0 + per : rows;
    float aw = 0.f, ab = 0.f;
    for (long long r = r0; r < r1; ++r) {
        const float g = to_f32(dy[r * D + c]);
        aw += g * (to_f32(s[r * D + c]) - mean[r]) * rstd[r];
        ab += g;
    }
    part[(size_t)blockIdx.y * 2 * D + c] = aw;
    part[(size_t)blockIdx.y * 2 * D + D + c] = ab;
}

// dw / db = the partial rows added in order: 32 columns per workgroup, 32 threads per column, each over every 32nd row,
// joined through LDS
__global__ __launch_bounds__(1024) void norm_fold_kernel(const float* __restrict__ part, int nparts, int D,
                                                         float* __restrict__ dw, float* __restrict__ db) {
    __shared__ float sm[32][33];
    const int cx = threadIdx.x & 31, py = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + cx;
    float a = 0.f;
    if (c < 2 * D) {
#pragma unroll 8
        for (int p = py; p < nparts; p += 32) a += part[(size_t)p * 2 * D + c];
    }
    sm[py][cx] = a;
    __syncthreads();
    if (py == 0 && c < 2 * D) {
#pragma unroll
        for (int k = 1; k < 32; ++k) a += sm[k][cx];
        if (c < D) {
            if (dw) dw[c] = a;
        } else if (db) {
            db[c - D] = a;
        }
    }
}

// Which lanes hold a row of D elements: G lanes with NC pieces of V elements each, at most 32 elements per
// lane (more and the backward pass, with four arrays of them, spills).  A wave or less while that is
// enough (a workgroup for 16 elements per lane and more was slower: bf16 rows of 2048 backward 61 us against 51), a
// workgroup up to D = 8192, wide = true beyond.
struct RowPlan { int G, NC, V; bool wide; };
RowPlan row_plan(int D, int dtype) {
    const int V = D >= (dtype == SF_BF16 ? 8 : 4) ? (dtype == SF_BF16 ? 8 : 4) : 1;
    const int pieces = (D + V - 1) / V;
    int G = 8;
    while (G < 64 && G < pieces) G *= 2;
    if (pieces > 64 * (32 / V)) G = NT;
    int NC = (pieces + G - 1) / G;
    if (NC == 5 || NC == 7) ++NC;
    return {G, NC, V, NC * V > 32};
}

// Persistent workgroups: four per CU keep the memory pipe full (two when a row takes the whole workgroup,
// whose partial rows are long)
int norm_grid(const RowPlan& p, long long rows) {
    const long long want = (rows + NT / p.G - 1) / (NT / p.G);
    const long long most = p.G == NT ? 512 : MAX_PARTS;
    return (int)(want < most ? want : most);
}

// calls f(G, NC, V, FULL) as integral constants for the plan of a row
template <typename T, typename F> bool with_plan(const RowPlan& p, int D, F&& f) {
    constexpr int V = ElemTraits<T>::EPC;
#define SF_PLAN(g, n, v)                                                                                                    \
    if (p.G == g && p.NC == n && p.V == v) {                                                                                \
        const std::integral_constant<int, g> G_;                                                                            \
        const std::integral_constant<int, n> N_;                                                                            \
        const std::integral_constant<int, v> V_;                                                                            \
        if (D == g * n * v) f(G_, N_, V_, std::true_type{});                                                                \
        else f(G_, N_, V_, std::false_type{});                                                                              \
        return true;                                                                                                        \
    }
    SF_PLAN(8, 1, 1)
    SF_PLAN(8, 1, V) SF_PLAN(16, 1, V) SF_PLAN(32, 1, V)
    SF_PLAN(64, 1, V) SF_PLAN(64, 2, V) SF_PLAN(64, 3, V) SF_PLAN(64, 4, V)
    SF_PLAN(NT, 3, V) SF_PLAN(NT, 4, V)
    if constexpr (V == 8) { SF_PLAN(NT, 2, V) }
    if constexpr (V == 4) { SF_PLAN(64, 6, V) SF_PLAN(64, 8, V) SF_PLAN(NT, 6, V) SF_PLAN(NT, 8, V) }
#undef SF_PLAN
    return false;
}

template <typename T>
int norm_fwd(const void* x, const void* res, void* sum, const float* w, const float* b, void* y, float* mean, float* rstd,
             long long rows, int D, float eps, hipStream_t st) {
    const RowPlan p = row_plan(D, ElemTraits<T>::CODE);
    if (p.wide) {
        const int grid = (int)(rows < 2048 ? rows : 2048);
        hipLaunchKernelGGL((norm_fwd_wide_kernel<T>), dim3(grid), dim3(NT), 0, st, (const T*)x, (const T*)res, (T*)sum, w, b,
                           (T*)y, mean, rstd, rows, D, eps);
    } else {
        const bool found = with_plan<T>(p, D, [&](auto g, auto n, auto v, auto full) {
            hipLaunchKernelGGL((norm_fwd_kernel<T, g.value, n.value, v.value, full.value>), dim3(norm_grid(p, rows)), dim3(NT), 0, st,
                               (const T*)x, (const T*)res, (T*)sum, w, b, (T*)y, mean, rstd, rows, D, eps);
        });
        SF_REQUIRE(found, "sf_layer_norm_fwd: no kernel for D = %d", D);
    }
    SF_LAUNCH_CHECK("sf_layer_norm_fwd");
    return SF_OK;
}

// rows of partial sums a backward call writes
int norm_parts(const RowPlan& p, long long rows) {
    if (!p.wide) return norm_grid(p, rows);
    return (int)(rows < 64 ? rows : 64);
}

template <typename T>
int norm_bwd(const void* dy, const void* dsum, const void* s, const float* w, const float* mean, const float* rstd, void* dx,
             float* dw, float* db, float* part, long long rows, int D, hipStream_t st) {
    const RowPlan p = row_plan(D, ElemTraits<T>::CODE);
    const int nparts = norm_parts(p, rows);
    float* const pw = dw || db ? part : nullptr;
    if (p.wide) {
        const int grid = (int)(rows < 2048 ? rows : 2048);
        hipLaunchKernelGGL((norm_bwd_wide_kernel<T>), dim3(grid), dim3(NT), 0, st, (const T*)dy, (const T*)dsum, (const T*)s, w,
                           mean, rstd, (T*)dx, rows, D);
        if (pw)
            hipLaunchKernelGGL((norm_bwd_cols_kernel<T>), dim3(ceil_div(D, NT), nparts), dim3(NT), 0, st, (const T*)dy,
                               (const T*)s, mean, rstd, pw, rows, (rows + nparts - 1) / nparts, D);
    } else {
        const bool found = with_plan<T>(p, D, [&](auto g, auto n, auto v, auto full) {
            hipLaunchKernelGGL((norm_bwd_kernel<T, g.value, n.value, v.value, full.value>), dim3(nparts), dim3(NT), 0, st, (const T*)dy,
                               (const T*)dsum, (const T*)s, w, mean, rstd, (T*)dx, pw, rows, D);
        });
        SF_REQUIRE(found, "sf_layer_norm_bwd: no kernel for D = %d", D);
    }
    SF_LAUNCH_CHECK("sf_layer_norm_bwd");
    if (pw) {
        hipLaunchKernelGGL(norm_fold_kernel, dim3(ceil_div(2LL * D, 32)), dim3(1024), 0, st, pw, nparts, D, dw, db);
        SF_LAUNCH_CHECK("sf_layer_norm_bwd (fold)");
    }
    return SF_OK;
}

}  // namespace

extern "C" int sf_layer_norm_fwd(const void* x, const void* residual, void* sum, const float* w, const float* b, void* y,
                                 float* mean, float* rstd, long long rows, int D, float eps, int dtype, void* stream) {
    SF_REQUIRE(dtype == SF_F32 || dtype == SF_BF16, "sf_layer_norm_fwd: unknown dtype %d", dtype);
    SF_REQUIRE(x && y && rows > 0 && D > 0 && D <= SF_NORM_MAX_DIM, "sf_layer_norm_fwd: bad arguments (rows %lld, D %d)", rows, D);
    SF_REQUIRE(!residual == !sum, "sf_layer_norm_fwd: residual and sum go together");
    SF_REQUIRE(!mean == !rstd, "sf_layer_norm_fwd: mean and rstd go together");
    SF_REQUIRE(eps >= 0.f, "sf_layer_norm_fwd: eps must not be negative");
    return dtype == SF_BF16 ? norm_fwd<bf16>(x, residual, sum, w, b, y, mean, rstd, rows, D, eps, (hipStream_t)stream)
                            : norm_fwd<float>(x, residual, sum, w, b, y, mean, rstd, rows, D, eps, (hipStream_t)stream);
}

extern "C" size_t sf_layer_norm_bwd_workspace_bytes(long long rows, int D, int dtype) {
    if (rows <= 0 || D <= 0 || D > SF_NORM_MAX_DIM || (dtype != SF_F32 && dtype != SF_BF16)) return 0;
    return (size_t)norm_parts(row_plan(D, dtype), rows) * 2 * D * sizeof(float);
}

extern "C" int sf_layer_norm_bwd(const void* dy, const void* dsum, const void* s, const float* w, const float* mean,
                                 const float* rstd, void* dx, float* dw, float* db, void* ws, size_t ws_bytes, long long rows,
                                 int D, int dtype, void* stream) {
    SF_REQUIRE(dtype == SF_F32 || dtype == SF_BF16, "sf_layer_norm_bwd: unknown dtype %d", dtype);
    SF_REQUIRE(dy && s && mean && rstd && dx && rows > 0 && D > 0 && D <= SF_NORM_MAX_DIM,
               "sf_layer_norm_bwd: bad arguments (rows %lld, D %d)", rows, D);
    SF_REQUIRE(!(dw || db) || (ws && ws_bytes >= sf_layer_norm_bwd_workspace_bytes(rows, D, dtype)),
               "sf_layer_norm_bwd: workspace of %zu bytes is too small (%zu)", ws_bytes,
               sf_layer_norm_bwd_workspace_bytes(rows, D, dtype));
    return dtype == SF_BF16 ? norm_bwd<bf16>(dy, dsum, s, w, mean, rstd, dx, dw, db, (float*)ws, rows, D, (hipStream_t)stream)
                            : norm_bwd<float>(dy, dsum, s, w, mean, rstd, dx, dw, db, (float*)ws, rows, D, (hipStream_t)stream);
}
