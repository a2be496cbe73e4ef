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
// enter the second product (bf16: at most half a step, 2^-8 of each, the size of the inputs' own rounding; relative to
// its norm the output is then 2.2e-3 off and the gradients of q and k 2.6e-3 to 2.9e-3, where rounding the exact result to bf16
// costs 1.7e-3).  The f32 form runs through the same code with f32 matrix instructions and rounds nothing.
//
// Layout.  Heads are [.., 2, d] rows (v and o: [.., 2 d], treated as two halves as well), d <= 64 a multiple of 8,
// padded to DP = 16, 32 or 64 columns per half inside a tile.  A tile in LDS is [row][2 DP] and is read in two ways: 32 rows
// at one 16-byte piece (an operand whose reduction axis is the columns) and 8 rows at 32 columns (reduction over the
// rows, through the transposing LDS read).  Tiles arrive by buffer loads that write LDS directly; pieces outside
// a sample's rows or a head's columns are out of the buffer's range and arrive as zeros, so keys
// behind a sample's length are never read.  Accumulators hold [reduction-free axis of the second product] x
// [query or key], so that the query's (key's) softmax state and scale are one register per lane and the
// probabilities leave the first product in the very registers the second one reads (the reduction axis is permuted
// the same way in both of its operands).
#include "sf_common.h"
#include "../../include/sfhip.h"

namespace {

// LDS is addressed through 32-bit pointers of its own address space throughout: with generic ones the constant parts of the
// tile addresses do not reach the instructions' offset fields, and every address takes a register.
#define SF_LDS __attribute__((address_space(3)))
typedef SF_LDS char* lds_ptr;
typedef const SF_LDS char* lds_cptr;

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
// Rows of NCH 16-byte pieces.  A copy instruction of a wave fills 1 KB, GROUP rows; groups are shifted against each other
// (pad) and the pieces of a row XORed (x), so that both 16 rows at one piece and 4 rows at 64 bytes cover the 256-byte
// bank window once.  XOR and shift touch few bits on purpose: the rest of an address is a constant of the instruction,
// and a lane needs 4 address registers for its row pieces and 4 for its column pieces (a full XOR of the piece index takes
// 8 and 8), or 2 and 2 from which one instruction makes each of the four (Lane).
template <typename T, int DP> struct Tile {
    static constexpr int EPC = 16 / (int)sizeof(T);       // elements per 16-byte piece
    static constexpr int NCH = 2 * DP / EPC;
    static constexpr int ROWB = NCH * 16;
    static constexpr int GROUP = 1024 / ROWB;
    static constexpr int XM = NCH == 32 ? 8 : NCH == 16 ? 12 : NCH == 8 ? 5 : 3;      // bits of the piece index that are XORed
    static __host__ __device__ __forceinline__ constexpr int x(int row) {
        return NCH == 32 ? (row & 1) << 3 : NCH == 16 ? (row & 3) << 2
               : NCH == 8 ? (((row >> 1) & 1) << 2) | ((row >> 2) & 1) : (row >> 2) & 3;
    }
    static __host__ __device__ __forceinline__ constexpr int pad(int g) { return NCH >= 16 ? g * 16 : NCH == 8 ? g * 32 : 0; }
    static __host__ __device__ __forceinline__ constexpr int row_off(int row) { return row * ROWB + pad(row / GROUP); }
    static constexpr int bytes(int rows) { return row_off(rows); }
    // A lane's share of the byte offset of piece c_const + c_lane of row r_const + r_lane (rows and pieces: no common bits of the
    // two, the shift and the XOR of the sum are those of its terms)
    struct Lane { int part, mix; };
    static __device__ __forceinline__ Lane lane_at(int r_lane, int c_lane, int byte) {
        return {row_off(r_lane) + ((c_lane & ~XM) << 4) + byte, ((c_lane & XM) ^ x(r_lane)) << 4};
    }
    static __device__ __forceinline__ int at(Lane l, int r_const, int c_const) {
        return (l.part + (l.mix ^ (((c_const & XM) ^ x(r_const)) << 4))) + (row_off(r_const) + ((c_const & ~XM) << 4));
    }
    static __device__ __forceinline__ Lane row_lane(int lane) { return lane_at(lane & 31, (lane >> 5) * (8 / EPC), 0); }
    static __device__ __forceinline__ Lane col_lane(int lane) {
        const int h = lane >> 5, i = lane & 15;
        if constexpr (sizeof(T) == 2) return lane_at(4 * h + (i >> 2), 2 * ((lane >> 4) & 1) + ((i & 3) >> 1), (i & 1) * 8);
        else return lane_at(4 * h, (lane & 31) >> 2, (lane & 3) * 4);
    }
    // columns 16 n + 8 h .. + 7 of row r_const + lane % 32, h = lane / 32 (r_const a multiple of 32)
    static __device__ __forceinline__ Frag<T> row_piece(lds_cptr t, Lane l, int r_const, int n) {
        Frag<T> f;
        if constexpr (sizeof(T) == 2) {
            f.v = *(const SF_LDS bf16x8*)(t + at(l, r_const, 2 * n));
        } else {
            const f32x4 lo = *(const SF_LDS f32x4*)(t + at(l, r_const, 4 * n));
            const f32x4 hi = *(const SF_LDS f32x4*)(t + at(l, r_const, 4 * n + 1));
#pragma unroll
            for (int j = 0; j < 4; ++j) { f.v[j] = lo[j]; f.v[4 + j] = hi[j]; }
        }
        return f;
    }
    // column 32 n + lane % 32 of rows r_const + acc_row(0..7, lane / 32) (r_const a multiple of 16): the reduction axis is the
    // rows, in the order the accumulators hold them
    static __device__ __forceinline__ Frag<T> col_piece(lds_cptr t, Lane l, int r_const, int n) {
        Frag<T> f;
        if constexpr (sizeof(T) == 2) {
            const bf16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((SF_LDS bf16x4*)(t + at(l, r_const, 4 * n)));
            const bf16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((SF_LDS bf16x4*)(t + at(l, r_const + 8, 4 * n)));
#pragma unroll
            for (int j = 0; j < 4; ++j) { f.v[j] = a[j]; f.v[4 + j] = b[j]; }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) f.v[j] = *(const SF_LDS float*)(t + at(l, r_const + acc_row(j, 0), 8 * n));
        }
        return f;
    }
};

// 64 lanes x 16 bytes from the buffer's byte offsets `off` + `soff` to LDS from `dst` on (uniform); zeros where off lies outside
// the buffer.  (Not in a template: in one, the host pass drops the launch stubs of every kernel that uses the builtin.)
__device__ __forceinline__ void copy_piece(__amdgpu_buffer_rsrc_t rs, lds_ptr dst, int off, int soff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, dst, 16, off, soff, 0, 0);
}

// Copies ROWS rows of a [.., 2, d] array into a tile, NW waves together, STEP rows at a time.  A lane's byte offset is the
// same in every step of every tile (the XOR of a row's pieces repeats every STEP rows); the step's first row enters
// through the buffer's base address (64 bits).
template <typename T, int DP, int ROWS, int NW> struct Copy {
    using L = Tile<T, DP>;
    static constexpr int STEP = NW * L::GROUP < ROWS ? NW * L::GROUP : ROWS;
    static_assert(ROWS % STEP == 0 && (STEP % 16 == 0 || L::x(STEP) == L::x(0)), "whole steps that repeat the XOR");
    int off, stride, row_bytes;         // bytes
    __device__ __forceinline__ Copy(long long stride_elems, int d) {
        stride = (int)(stride_elems * (long long)sizeof(T));
        row_bytes = 2 * d * (int)sizeof(T);
        const int i = threadIdx.x, row = i / L::NCH, piece = (i % L::NCH) ^ L::x(row);
        const int half = piece / (L::NCH / 2), e = (piece % (L::NCH / 2)) * L::EPC;
        off = e < d ? row * stride + (half * d + e) * (int)sizeof(T) : (int)0x80000000;
    }
    // ROWS rows from `p` on, of which the first `have` exist.  A whole tile takes one buffer, the steps being scalar offsets;
    // at the end of the rows every step gets a buffer of its own.  (Offsets stay below 2^32: 128 rows of less than 2^24 bytes.)
    __device__ __forceinline__ void issue(const T* p, int have, lds_ptr dst) const {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        if (wave * L::GROUP >= STEP) return;
        dst += L::row_off(wave * L::GROUP);
        if (have >= ROWS) {
            const __amdgpu_buffer_rsrc_t rs =
                __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (unsigned)(ROWS - 1) * (unsigned)stride + (unsigned)row_bytes, 0x00020000);
#pragma unroll
            for (int r = 0; r < ROWS; r += STEP) copy_piece(rs, dst + L::row_off(r), off, r * stride);
        } else {
#pragma unroll
            for (int r = 0; r < ROWS; r += STEP) {
                const int n = min(have - r, STEP);
                const unsigned bytes = n > 0 ? (unsigned)(n - 1) * (unsigned)stride + (unsigned)row_bytes : 0u;
                const __amdgpu_buffer_rsrc_t rs =
                    __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)p + (long long)r * stride), 0, bytes, 0x00020000);
                copy_piece(rs, dst + L::row_off(r), off, 0);
            }
        }
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

// Exponentials of a row are taken relative to a score `ref` that it has seen, and are 2^exponent(s), c being the scale in base 2.
// Scores may be of any finite size, so nothing may depend on c s as such: rounded to f32 it is off by half a step, 0.004 at
// 2^16, 1 at 2^24, 2^86 at 2^110.  While c ref is below FAR, the exponent is fma(s, c, -fl(c ref)), one rounding of its own
// size; that c ref was rounded is a factor between 2^-1/2 and 2^1/2 that all of the row's terms and their sum share.
// Beyond, no f32 lies near c ref any more, and the exponent is (s - ref) c: two roundings of its own size.  Which of
// the two it is depends on `ref` alone, so equal scores have equal terms wherever they are formed.
constexpr float FAR = 16777216.f;
__device__ __forceinline__ float scaled(float ref, float c) {
#pragma clang fp contract(off)
    return ref * c;
}
__device__ __forceinline__ bool is_far(float ref, float c) { return !(fabsf(scaled(ref, c)) < FAR); }
struct Exponent {
    float sub, neg;
    __device__ __forceinline__ Exponent(float ref, float c) {
        const bool far = is_far(ref, c);
        sub = far ? ref : 0.f;
        neg = far ? 0.f : -scaled(ref, c);
    }
    __device__ __forceinline__ float operator()(float s, float c) const { return fmaf(s - sub, c, neg); }
};
// 2^this takes terms relative to `from` to terms relative to `to`
__device__ __forceinline__ float change(float from, float to, float c) {
#pragma clang fp contract(off)
    const float far = -Exponent(from, c)(to, c), near = scaled(from, c) - scaled(to, c), between = fmaf(from, c, -scaled(to, c));
    return is_far(to, c) ? far : is_far(from, c) ? between : near;
}
// The backward pass takes probabilities as 2^(c s - lse), lse = c ref + log2(sum) in one f32, where every |lse| of a tile is below
// NEAR: off by 2^-18 of themselves at most.  Elsewhere as 2^(c (s - ref) - lg), one operation more; lg is log2(sum), less what the
// rounding of c ref has left in the sum.
constexpr float NEAR = 64.f;

// a row's reference before it has seen a key: no finite score is below it, and it is itself finite, so that its differences
// with masked scores (-inf) and with other references are never NaN
constexpr float NO_SCORE = -3.4028234663852886e38f;

// waves per SIMD that a kernel's registers have to leave room for: two, so that one computes while the other loads, but where the
// accumulators and f32 operands of 2 x 64 columns alone are more than half of them
template <typename T, int DP> constexpr int WAVES = sizeof(T) == 4 && DP == 64 ? 1 : 2;

struct Strides { long long b, t, h; };      // elements
template <typename T> struct Args {
    const T* q; const T* k; const T* v;
    Strides qs, ks, vs;
    const void* lam;
    const int* lengths;
    T* o; float* maps; float* sums;         // maps f32 [B,Tq,H,2,2d] = O_1, O_2; sums f32 [B,H,Tq,2,2] = (ref, sum) of each map: for the backward pass
    float* part;                            // partial results of the work items that are cut
    const T* dout; const float* maps_in; const float* sums_in;
    float* stat;                            // [B,H,STATS,Tp], see attn_delta_kernel; zeros from Tq to Tp
    T* dq; T* dk; T* dv;
    int lam_bf16, B, Tq, Tp, Tk, H, Hk, d, causal;        // Tp: Tq rounded up to whole tiles of any kernel
    int full, parts;                        // see Cut
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

// Work items (a tile of rows or keys of one batch and key/value head) below `full` go to one workgroup each, the others to
// `parts` workgroups that share out the item's tiles of the other axis; their partial results are joined by a second launch.
struct Work { int item, part, parts, tail; };
__device__ __forceinline__ Work work_of(int id, int full, int parts) {
    if (id < full) return {id, 0, 1, 0};
    const int e = id - full;
    return {full + e / parts, e % parts, parts, e / parts};
}
// Work item -> (batch and key/value head, tile).  Ids go round the 8 XCDs.  Items of equal length: when the heads divide by 8,
// all the tiles of a head stay on one XCD, whose L2 then holds what they share.  Causal items get shorter with the tile
// index: longest first, every other 256 in reverse, so that the workgroups that meet on a CU make up for each other.
__device__ __forceinline__ void locate(int id, int heads, int tiles, int causal, int& bh, int& x) {
    if (causal) {
        const int j = id & 255;
        if ((id & 256) && (id | 255) < heads * tiles) id = (id & ~255) + (31 - (j >> 3)) * 8 + (j & 7);
        bh = id % heads;
        x = id / heads;
    } else if (heads % 8 == 0) {
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

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
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
// all keys of the tile.  KEYS_SPLIT true (single tokens, and wherever row_plan finds the wider items too few): all waves take the
// same 32 rows and wave w the keys 32 w .. of the tile; the waves' results are joined through LDS at the end.
// Measured, bf16 heads of 2 x 64: 8 heads, 2 x 5120 tokens: 340 to 375 us, 322 GFLOP, 0.9 PFLOP/s (a library product reaches 1.28);
// the matrix pipe is busy 47 % of the time and the vector unit (32 exponentials a lane and tile of 32 x 32) nearly as long, hardly
// at the same time, at a clock that power holds at 1.75 GHz.  1 x 8191 tokens, causal: 262 to 280 us, 206 GFLOP.  Single tokens,
// 16 samples, 4 key heads, 8192 keys: 30 us, 134 MB, 4.4 TB/s, bound by HBM.
// (narrow heads: four waves per SIMD, as many as slots_of counts on)
template <typename T, int DP, int NW, bool KEYS_SPLIT, int KT>
__global__ __launch_bounds__(64 * NW, (DP == 16 && !KEYS_SPLIT ? 4 : WAVES<T, DP>)) void attn_fwd_kernel(Args<T> a) {
    using L = Tile<T, DP>;
    constexpr int KS = DP / 16, DT = 2 * DP / 32;
    constexpr int RB = KEYS_SPLIT ? 32 : 32 * NW;
    constexpr int TB = L::bytes(KT);                       // of a key or value tile
    extern __shared__ __align__(16) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h2 = lane >> 5;
    const int group = a.H / a.Hk;
    const long long rows = (long long)group * a.Tq;
    const int tiles = (int)((rows + RB - 1) / RB);
    const Work w = work_of(blockIdx.x, a.full, a.parts);
    int bh, x;
    locate(w.item, a.B * a.Hk, tiles, a.causal, bh, x);
    const int rt = tiles - 1 - x;                          // causal rows see more keys the later they are
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
    const int all = (kstop + KT - 1) / KT, per = (all + w.parts - 1) / w.parts;
    const int first = w.part * per, last = min(all, first + per);

    Frag<T> qf[2][KS];
    const T* qrow = a.q + b * a.qs.b + t * a.qs.t + hq * a.qs.h;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[i][s] = global_piece<T>(qrow, i, s * 16 + 8 * h2, a.d, true);

    f32x16 acc[2][DT];
    float ref[2], l[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        ref[i] = NO_SCORE;
        l[i] = 0.f;
#pragma unroll
        for (int n = 0; n < DT; ++n) acc[i][n] = zero16();
    }
    const T* const kbase = a.k + b * a.ks.b + hk * a.ks.h;
    const T* const vbase = a.v + b * a.vs.b + hk * a.vs.h;
    const Copy<T, DP, KT, NW> kc(a.ks.t, a.d), vc(a.vs.t, a.d);
    lds_ptr const buf0 = (lds_ptr)smem;
    lds_ptr const buf1 = buf0 + 2 * TB;

    const typename L::Lane rl = L::row_lane(lane), cl = L::col_lane(lane);

    auto sub_tile = [&](lds_cptr kt, lds_cptr vt, int sub, int key0) {
        if (key0 >= vmax) return;
        f32x16 s[2] = {zero16(), zero16()};
#pragma unroll
        for (int n = 0; n < KS; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                s[i] = mma(L::row_piece(kt, rl, sub, i * KS + n), qf[i][n], s[i]);
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
            // The reference of the exponentials only has to keep them in range: it moves when a lane's 16 of them add up to more
            // than 2^12, then to the row's maximum.  The usual tile so needs no maximum, no exchange between lanes
            // and no rescaling.  Where a row has seen no key yet, or its reference is far, the attempt does not count (it is made
            // all the same: behind a branch it could not overlap with the products).
            float p[16], sum = 0.f;
            const float at = scaled(ref[i], a.c);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                p[r] = __builtin_amdgcn_exp2f(fmaf(s[i][r], a.c, -at));
                sum += p[r];
            }
            if (__any((sum > 4096.f) | !(fabsf(at) < FAR))) {
                float top = s[i][0];
#pragma unroll
                for (int r = 1; r < 16; ++r) top = fmaxf(top, s[i][r]);
                const float to = fmaxf(ref[i], fmaxf(top, __shfl_xor(top, 32, 64))), f = exp2f(change(ref[i], to, a.c));
                ref[i] = to;
                l[i] *= f;
#pragma unroll
                for (int n = 0; n < DT; ++n)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[i][n][r] *= f;
                __builtin_amdgcn_sched_barrier(0);         // (fewer registers)
                sum = 0.f;
                const Exponent exponent(to, a.c);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    p[r] = __builtin_amdgcn_exp2f(exponent(s[i][r], a.c));
                    sum += p[r];
                }
            }
            l[i] += sum;
            pack(pf[i][0], p);
            pack(pf[i][1], p + 8);
        }
#pragma unroll
        for (int n = 0; n < DT; ++n)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const Frag<T> vf = L::col_piece(vt, cl, sub + 16 * u, n);
                acc[0][n] = mma(vf, pf[0][u], acc[0][n]);
                acc[1][n] = mma(vf, pf[1][u], acc[1][n]);
            }
    };
    // `cur` holds tile i, `fill` takes tile i + 1 (restrict: the reads need not wait for that copy)
    auto step = [&](int i, lds_cptr __restrict__ cur, lds_ptr __restrict__ fill) {
        if (i + 1 < last) {
            kc.issue(kbase + (i + 1) * KT * a.ks.t, kend - (i + 1) * KT, fill);
            vc.issue(vbase + (i + 1) * KT * a.vs.t, kend - (i + 1) * KT, fill + TB);
        }
        if constexpr (KEYS_SPLIT) {
            sub_tile(cur, cur + TB, wave * 32, i * KT + wave * 32);
        } else {
#pragma unroll
            for (int u = 0; u < KT / 32; ++u) sub_tile(cur, cur + TB, u * 32, i * KT + u * 32);
        }
    };
    if (first < last) {
        kc.issue(kbase + first * KT * a.ks.t, kend - first * KT, buf0);
        vc.issue(vbase + first * KT * a.vs.t, kend - first * KT, buf0 + TB);
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
        float* const box = reinterpret_cast<float*>(smem);             // [2 DT 16][64] accumulators, then ref, l
#pragma unroll 1
        for (int u = 1; u < NW; ++u) {
            __syncthreads();
            if (wave == u) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
#pragma unroll
                    for (int n = 0; n < DT; ++n)
#pragma unroll
                        for (int r = 0; r < 16; ++r) box[((i * DT + n) * 16 + r) * 64 + lane] = acc[i][n][r];
                    box[(2 * DT * 16 + 2 * i) * 64 + lane] = ref[i];
                    box[(2 * DT * 16 + 2 * i + 1) * 64 + lane] = l[i];
                }
            }
            __syncthreads();
            if (wave == 0) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float other = box[(2 * DT * 16 + 2 * i) * 64 + lane], lo = box[(2 * DT * 16 + 2 * i + 1) * 64 + lane];
                    const float to = fmaxf(ref[i], other), f = exp2f(change(ref[i], to, a.c)), g = exp2f(change(other, to, a.c));
                    ref[i] = to;
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
    if (w.parts > 1) {
        const long long at = ((long long)w.tail * w.parts + w.part) * RB + (row - r0);
        const long long items = (gridDim.x - a.full) / a.parts;
        float* const po = a.part + at * (4 * DP);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int n = 0; n < DT; ++n)
#pragma unroll
                for (int r = 0; r < 16; r += 4)
                    *reinterpret_cast<float4*>(po + i * 2 * DP + 32 * n + acc_row(r, h2)) =
                        float4{acc[i][n][r], acc[i][n][r + 1], acc[i][n][r + 2], acc[i][n][r + 3]};
        if (h2 == 0)
            *reinterpret_cast<float4*>(a.part + items * w.parts * RB * (4 * DP) + at * 4) = float4{ref[0], l[0], ref[1], l[1]};
        return;
    }
    // a row that sees no key has l = 0: its output is zero
    const float i1 = l[0] > 0.f || l[0] != l[0] ? 1.f / l[0] : 0.f, i2 = l[1] > 0.f || l[1] != l[1] ? 1.f / l[1] : 0.f;
    const float lam = lam_of(a.lam, a.lam_bf16, hq);
    const long long out = (((long long)b * a.Tq + t) * a.H + hq) * (2 * a.d);
#pragma unroll
    for (int n = 0; n < DT; ++n)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            float x1[4], y[4], z[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x1[e] = acc[0][n][r + e] * i1;
                z[e] = acc[1][n][r + e] * i2;
                y[e] = fmaf(-lam, z[e], x1[e]);        // (spelled out: the same bits with and without the maps)
            }
            store_cols<T, DP>(a.o + out, 32 * n + acc_row(r, h2), a.d, y[0], y[1], y[2], y[3]);
            if (a.maps) {
                const int c = 32 * n + acc_row(r, h2);
                store_cols<float, DP>(a.maps + 2 * out, c, a.d, x1[0], x1[1], x1[2], x1[3]);
                store_cols<float, DP>(a.maps + 2 * out + 2 * a.d, c, a.d, z[0], z[1], z[2], z[3]);
            }
        }
    if (a.sums && h2 == 0) *reinterpret_cast<float4*>(a.sums + (((long long)b * a.H + hq) * a.Tq + t) * 4) = float4{ref[0], l[0], ref[1], l[1]};
}

// joins the parts of the forward items that were cut: one wave per query row (2 x 5120 tokens, two parts for a fifth of the rows:
// 18 us; single tokens of 64 key heads, four parts: 6 us)
template <typename T, int DP> __global__ __launch_bounds__(256) void attn_join_kernel(Args<T> a, int rb, int items) {
    const int lane = threadIdx.x & 63;
    const int group = a.H / a.Hk;
    const long long rows = (long long)group * a.Tq, id = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int tail = (int)(id / rb), tiles = (int)((rows + rb - 1) / rb);
    if (tail >= items) return;
    int bh, x;
    locate(a.full + tail, a.B * a.Hk, tiles, a.causal, bh, x);
    const long long row = (long long)(tiles - 1 - x) * rb + id % rb;
    if (row >= rows) return;
    const int b = bh / a.Hk, t = (int)(row / group), hq = bh % a.Hk * group + (int)(row % group);
    const long long at0 = (long long)tail * a.parts * rb + id % rb;
    // lane s holds the state of part s (there are at most 64)
    const float* const pm = a.part + (long long)items * a.parts * rb * (4 * DP);
    float4 v{NO_SCORE, 0.f, NO_SCORE, 0.f};
    if (lane < a.parts) v = *reinterpret_cast<const float4*>(pm + (at0 + (long long)lane * rb) * 4);
    const float ref[2] = {wave_max(v.x), wave_max(v.z)};
    const float f1 = exp2f(change(v.x, ref[0], a.c)), f2 = exp2f(change(v.z, ref[1], a.c));
    const float l[2] = {wave_sum(v.y * f1), wave_sum(v.w * f2)};
    constexpr int NCOL = (2 * DP + 63) / 64;
    float acc[2][NCOL];
#pragma unroll
    for (int n = 0; n < NCOL; ++n) acc[0][n] = acc[1][n] = 0.f;
#pragma unroll 4
    for (int s = 0; s < a.parts; ++s) {
        const float* const po = a.part + (at0 + (long long)s * rb) * (4 * DP);
        const float w1 = __shfl(f1, s, 64), w2 = __shfl(f2, s, 64);
#pragma unroll
        for (int n = 0; n < NCOL; ++n) {
            const int c = n * 64 + lane;
            if (c < 2 * DP) {
                acc[0][n] += po[c] * w1;
                acc[1][n] += po[2 * DP + c] * w2;
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
        const float x1 = acc[0][n] * i1, z = acc[1][n] * i2;
        a.o[out + half * a.d + j] = from_f32<T>(fmaf(-lam, z, x1));
        if (a.maps) {
            a.maps[2 * out + half * a.d + j] = x1;
            a.maps[2 * out + (2 + half) * a.d + j] = z;
        }
    }
    if (a.sums && lane == 0) *reinterpret_cast<float4*>(a.sums + (((long long)b * a.H + hq) * a.Tq + t) * 4) = float4{ref[0], l[0], ref[1], l[1]};
}

// ------------------------------------------------------------------------------ backward
constexpr int STATS = 9;                // values of a row

// stat = lse_1, -delta_1, lse_2, lam (delta_2 - delta_1), ref_1, lg_1, ref_2, lg_2, delta_2 of every row; delta_i = do . O_i
// (the last one is for dlam alone, and in bf16 the query gradients' kernel writes a better one).  A row that saw no key gets infinite lse
// and ref, which make its probabilities zero.  16 lanes per row.  What the two
// gradient kernels would compute for every score is in them: -delta_1 starts the accumulators of dP, so that
// dP - delta_1 costs nothing, and -lam (dP - delta_2) is one multiply-add from it (2 x 5120 tokens, 8 heads: dq 384 to
// 372 us, dk and dv 597 to 589).  O_1 and O_2 are kept in f32: the gradients of the scores are differences dP - delta,
// and rounding the maps to bf16 as well raises the relative error of dq from 2.9e-3 to 3.6e-3 (32 x 365 tokens).  Bound by HBM:
// 24 us for the 210 MB of 2 x 5120 tokens and 8 heads of 2 x 64, most of it the maps.
template <typename T> __global__ __launch_bounds__(256) void attn_delta_kernel(Args<T> a) {
    const long long id = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);       // (b, t, h), t up to Tp
    const int q = threadIdx.x & 15, h = (int)(id % a.H), t = (int)(id / a.H % a.Tp);
    const long long b = id / a.H / a.Tp;
    if (b >= a.B) return;
    float d1 = 0.f, d2 = 0.f;
    if (8 * q < 2 * a.d && t < a.Tq) {
        const long long row = ((b * a.Tq + t) * a.H + h) * (2 * a.d) + 8 * q, map = row * 2 - 8 * q;
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
            Vec4<T> g;
            Vec4<float> x, z;
            g.load(a.dout + row + j);
            x.load(a.maps_in + map + j);
            z.load(a.maps_in + map + 2 * a.d + j);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                d1 += g.get(e) * x.get(e);
                d2 += g.get(e) * z.get(e);
            }
        }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
        d1 += __shfl_xor(d1, o, 64);
        d2 += __shfl_xor(d2, o, 64);
    }
    if (q >= STATS) return;
    float v = q == 1 ? -d1 : q == 3 ? lam_of(a.lam, a.lam_bf16, h) * (d2 - d1) : d2;
    if (q != 1 && q != 3 && q != 8) {
        v = 0.f;
        if (t < a.Tq) {
            const float* const p = a.sums_in + ((b * a.H + h) * a.Tq + t) * 4 + (q == 2 || q > 5 ? 2 : 0);
            const float ref = p[0], sum = p[1], lg = sum > 0.f ? __log2f(sum) : sum;        // (0 stays 0, NaN NaN)
            if (q > 3 && q & 1) v = is_far(ref, a.c) ? lg : lg - fmaf(ref, a.c, -scaled(ref, a.c));
            else v = sum == 0.f ? INFINITY : q > 3 ? ref : scaled(ref, a.c) + lg;
        }
    }
    a.stat[((b * a.H + h) * STATS + q) * a.Tp + t] = v;
}

// dlam[h] = -sum over the rows of head h of delta_2, in 64 bits and a fixed order (10240 rows a head: 6 us, latency)
__global__ __launch_bounds__(1024) void attn_dlam_kernel(const float* __restrict__ stat, void* __restrict__ dlam, int lam_bf16,
                                                         int B, int H, int Tp) {
    __shared__ double sm[16];
    const int h = blockIdx.x;
    double s = 0.0;
    const long long n = (long long)B * Tp;
#pragma unroll 8
    for (long long i = threadIdx.x; i < n; i += 1024) s += (double)stat[((i / Tp * H + h) * STATS + STATS - 1) * Tp + i % Tp];
    s = wave_sum_d(s);
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 16; ++i) s += sm[i];
        if (lam_bf16) ((bf16*)dlam)[h] = (bf16)(float)-s;
        else ((float*)dlam)[h] = (float)-s;
    }
}

// adds the accumulators of waves 1 .. NW - 1 to those of wave 0, one wave after the other, through LDS (N * 1024 floats)
template <int NW, int N> __device__ __forceinline__ void join_waves(f32x16 (&acc)[N], float* box, int wave, int lane) {
#pragma unroll 1
    for (int u = 1; u < NW; ++u) {
        __syncthreads();
        if (wave == u) {
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) box[(n * 16 + r) * 64 + lane] = acc[n][r];
        }
        __syncthreads();
        if (wave == 0) {
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[n][r] += box[(n * 16 + r) * 64 + lane];
        }
    }
}

// Gradient of the queries: as the forward pass, rows (32 per wave) or the keys of a tile shared out.  (8 bf16 heads of 2 x 64, 2 x 5120 tokens:
// 350 to 390 us, 322 GFLOP, 0.86 PFLOP/s; bound as the forward pass.)
// bf16: delta_2 comes out of here again, as the sum of P_2 dP in f32, for dlam alone: over all the rows little is left of the terms of
// dlam, and with the delta_2 of the forward pass's bf16 probabilities it was off by 2e-3 to 4.5e-3 of itself.
template <typename T, int DP, int NW, bool KEYS_SPLIT, int KT>
__global__ __launch_bounds__(64 * NW, (WAVES<T, DP>)) void attn_dq_kernel(Args<T> a) {
    using L = Tile<T, DP>;
    constexpr int RB = KEYS_SPLIT ? 32 : 32 * NW, KS = DP / 16, VS = 2 * DP / 16;
    constexpr int NA = DP == 16 ? 2 : 2 * DP / 32;         // accumulators: 32 columns each (DP = 16: both halves in each)
    constexpr int TB = L::bytes(KT);
    extern __shared__ __align__(16) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h2 = lane >> 5;
    const int group = a.H / a.Hk;
    const long long rows = (long long)group * a.Tq;
    const int tiles = (int)((rows + RB - 1) / RB);
    const Work w = work_of(blockIdx.x, a.full, a.parts);
    int bh, x;
    locate(w.item, a.B * a.Hk, tiles, a.causal, bh, x);
    const int rt = tiles - 1 - x;
    const int b = bh / a.Hk, hk = bh % a.Hk;
    const long long r0 = (long long)rt * RB, row = r0 + (KEYS_SPLIT ? 0 : wave * 32) + (lane & 31);
    const bool have = row < rows;
    const long long rr = have ? row : rows - 1;
    const int t = (int)(rr / group), hq = hk * group + (int)(rr % group);
    const int kend = keys_of(a, b), reach = a.Tk - a.Tq;
    const int vis = a.causal ? max(0, min(kend, t + reach + 1)) : kend;
    const int vmin = wave_min_i(vis), vmax = wave_max_i(vis);
    const int t_last = (int)((r0 + RB < rows ? r0 + RB - 1 : rows - 1) / group);
    const int kstop = a.causal ? max(0, min(kend, t_last + reach + 1)) : kend;
    const int all = (kstop + KT - 1) / KT, per = (all + w.parts - 1) / w.parts;
    const int first = w.part * per, last = min(all, first + per);

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
    const float* const stat = a.stat + ((long long)b * a.H + hq) * STATS * a.Tp + t;
    float lse[2] = {stat[0], stat[2 * a.Tp]};              // or lg, with ref to be taken off the scores first
    const float apart = stat[3 * a.Tp], lam = lam_of(a.lam, a.lam_bf16, hq);
    const bool wide = __any(!(fmaxf(fabsf(lse[0]), fabsf(lse[1])) < NEAR));
    const float ref[2] = {stat[4 * a.Tp], stat[6 * a.Tp]};
    if (wide) {
        lse[0] = stat[5 * a.Tp];
        lse[1] = stat[7 * a.Tp];
    }
    f32x16 start;                                          // of dP - delta_1
#pragma unroll
    for (int r = 0; r < 16; ++r) start[r] = stat[a.Tp];
    f32x16 acc[NA];
#pragma unroll
    for (int n = 0; n < NA; ++n) acc[n] = zero16();
    constexpr bool SUM = sizeof(T) == 2;
    float p2dp = 0.f;                                      // sum of P_2 (dP - delta_1)
    const T* const kbase = a.k + b * a.ks.b + hk * a.ks.h;
    const T* const vbase = a.v + b * a.vs.b + hk * a.vs.h;
    const Copy<T, DP, KT, NW> kc(a.ks.t, a.d), vc(a.vs.t, a.d);
    lds_ptr const buf0 = (lds_ptr)smem;
    lds_ptr const buf1 = buf0 + 2 * TB;
    const typename L::Lane rl = L::row_lane(lane), cl = L::col_lane(lane);

    auto sub_tile = [&](lds_cptr kt, lds_cptr vt, int sub, int key0) {
        if (key0 >= vmax) return;
        f32x16 s[2] = {zero16(), zero16()}, dp = start;
#pragma unroll
        for (int n = 0; n < KS; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                s[i] = mma(L::row_piece(kt, rl, sub, i * KS + n), qf[i][n], s[i]);
#pragma unroll
        for (int n = 0; n < VS; ++n) dp = mma(L::row_piece(vt, rl, sub, n), gf[n], dp);
        if ((key0 + 32 > vmin) | wide) {        // (one branch: the usual tile takes none)
            if (key0 + 32 > vmin) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const bool see = key0 + acc_row(r, h2) < vis;
                    s[0][r] = see ? s[0][r] : -INFINITY;
                    s[1][r] = see ? s[1][r] : -INFINITY;
                }
            }
            if (wide) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    s[0][r] -= ref[0];
                    s[1][r] -= ref[1];
                }
            }
        }
        Frag<T> df[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float ds[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float y = __builtin_amdgcn_exp2f(fmaf(s[i][r], a.c, -lse[i]));
                if (SUM && i) p2dp = fmaf(y, dp[r], p2dp);
                ds[r] = y * (i ? fmaf(-lam, dp[r], apart) : dp[r]);
            }
            pack(df[i][0], ds);
            pack(df[i][1], ds + 8);
        }
#pragma unroll
        for (int n = 0; n < NA; ++n)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int map = DP == 16 ? n : 32 * n / DP;
                acc[n] = mma(L::col_piece(kt, cl, sub + 16 * u, DP == 16 ? 0 : n), df[map][u], acc[n]);
            }
    };
    auto step = [&](int i, lds_cptr __restrict__ cur, lds_ptr __restrict__ fill) {
        if (i + 1 < last) {
            kc.issue(kbase + (i + 1) * KT * a.ks.t, kend - (i + 1) * KT, fill);
            vc.issue(vbase + (i + 1) * KT * a.vs.t, kend - (i + 1) * KT, fill + TB);
        }
        if constexpr (KEYS_SPLIT) {
            sub_tile(cur, cur + TB, wave * 32, i * KT + wave * 32);
        } else {
#pragma unroll
            for (int u = 0; u < KT / 32; ++u) sub_tile(cur, cur + TB, u * 32, i * KT + u * 32);
        }
    };
    if (first < last) {
        kc.issue(kbase + first * KT * a.ks.t, kend - first * KT, buf0);
        vc.issue(vbase + first * KT * a.vs.t, kend - first * KT, buf0 + TB);
        for (int i = first;;) {
            stage_sync();
            step(i, buf0, buf1);
            if (++i >= last) break;
            stage_sync();
            step(i, buf1, buf0);
            if (++i >= last) break;
        }
    }
    if constexpr (KEYS_SPLIT) {
        join_waves<NW>(acc, (float*)smem, wave, lane);
        if constexpr (SUM) {
            float* const box = (float*)smem;
            __syncthreads();
            box[wave * 64 + lane] = p2dp;
            __syncthreads();
            for (int u = 1; u < NW; ++u)
                if (wave == 0) p2dp += box[u * 64 + lane];
        }
        if (wave != 0) return;
    }
    if constexpr (SUM) p2dp += __shfl_xor(p2dp, 32, 64);
    if (!have) return;
    if (SUM && h2 == 0) {
        const long long at = ((long long)w.tail * w.parts + w.part) * RB + (row - r0);
        if (w.parts > 1) a.part[(long long)(gridDim.x - a.full) * RB * (2 * DP) + at] = p2dp;
        else a.stat[(((long long)b * a.H + hq) * STATS + STATS - 1) * a.Tp + t] = p2dp - start[0];
    }
#pragma unroll
    for (int n = 0; n < NA; ++n)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int col = (DP == 16 ? 0 : 32 * n) + acc_row(r, h2), map = DP == 16 ? n : 32 * n / DP;
            if (col / DP != map) continue;
            const float4 y{acc[n][r] * a.scale, acc[n][r + 1] * a.scale, acc[n][r + 2] * a.scale, acc[n][r + 3] * a.scale};
            if (w.parts > 1)
                *reinterpret_cast<float4*>(a.part + (((long long)w.tail * w.parts + w.part) * RB + (row - r0)) * (2 * DP) + col) = y;
            else
                store_cols<T, DP>(a.dq + out, col, a.d, y.x, y.y, y.z, y.w);
        }
}

// Gradients of the keys and values: a wave owns 32 keys, the workgroup's 128 keys meet the query rows of every head of the
// group tile by tile.  SPLIT: the workgroup has 32 keys and the waves share out the rows of a tile; joined through LDS at the end.  The wave's keys stay in registers, the values in LDS.  bf16 heads of 2 x 64: with 128 accumulators and
// 32 registers of keys little is left of the 256 that two waves per SIMD have, and a spilled one is reloaded behind the copies
// under way.  So a lane keeps two address registers for its row pieces and two for its column pieces and makes the
// others where it uses them (fresh), and the maps come one after the other: no spill in the loop (2 x 5120 tokens, 8 heads:
// 725 us with 13 spills, 592 us without; eight waves in pairs, with the keys in LDS too, 635 us).  540 to 600 us now, 429 GFLOP,
// 0.75 PFLOP/s: the matrix pipe is busy 37 % of the time, LDS reads 33 %, and no registers are left to fetch operands ahead.
template <typename T, int DP, int NW, bool SPLIT>
__global__ __launch_bounds__(64 * NW, (WAVES<T, DP>)) void attn_dkv_kernel(Args<T> a) {
    using L = Tile<T, DP>;
    constexpr int KB = SPLIT ? 32 : 32 * NW, QT = SPLIT ? 32 * NW : 32, KS = DP / 16, VS = 2 * DP / 16, DT = 2 * DP / 32;
    constexpr int NA = DP == 16 ? 2 : DT;
    constexpr int TB = L::bytes(QT), SB = 32 * QT;         // query / gradient tile; row statistics, all but the last (copies of 1 KB)
    constexpr int BUF = 2 * TB + SB;
    extern __shared__ __align__(16) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h2 = lane >> 5;
    const int group = a.H / a.Hk;
    const int tiles = (a.Tk + KB - 1) / KB;
    const Work w = work_of(blockIdx.x, a.full, a.parts);
    int bh, x;
    locate(w.item, a.B * a.Hk, tiles, a.causal, bh, x);
    const int b = bh / a.Hk, hk = bh % a.Hk, k0 = x * KB;
    const int kw = SPLIT ? 0 : wave * 32, rows0 = SPLIT ? wave * 32 : 0;       // the wave's keys, and its rows of a tile
    const int key = k0 + kw + (lane & 31);
    const int kend = keys_of(a, b), reach = a.Tk - a.Tq;
    const int t_min = key >= kend ? 1 << 30 : a.causal ? key - reach : 0;  // the key is seen by queries from t_min on
    const int w_first = k0 + kw;                                    // the wave's first key
    const int w_tmax = a.causal ? w_first + 31 - reach : 0;                // queries from here on see all keys of the wave
    const int q_first = a.causal ? max(0, k0 - reach) / QT : 0;            // first query tile that sees a key of the workgroup
    const int q_tiles = (a.Tq + QT - 1) / QT;
    const int per_head = k0 < kend && q_first < q_tiles ? q_tiles - q_first : 0;
    const int all = per_head * group, per = (all + w.parts - 1) / w.parts;     // (head, query tile) pairs, head by head
    const int first = w.part * per, last = min(all, first + per);

    lds_ptr const buf0 = (lds_ptr)smem;                                    // (the buffers first: their addresses fit the offset fields)
    lds_ptr const buf1 = buf0 + BUF;
    lds_ptr const vmem = buf0 + 2 * BUF;                                   // [KB] value rows
    const T* const kbase = a.k + b * a.ks.b + hk * a.ks.h;
    const T* const vbase = a.v + b * a.vs.b + hk * a.vs.h;
    f32x16 dv[DT], dk[NA];
#pragma unroll
    for (int n = 0; n < DT; ++n) dv[n] = zero16();
#pragma unroll
    for (int n = 0; n < NA; ++n) dk[n] = zero16();

    const Copy<T, DP, QT, NW> q_copy(a.qs.t, a.d), g_copy((long long)a.H * 2 * a.d, a.d);
    const long long gstride = (long long)a.H * 2 * a.d;
    // the next tile to copy: (head, query tile) and where it lies
    struct Pos { int head, tile; const T* q; const T* g; const float* stat; } pos{};
    auto go_to = [&](int head, int tile) {
        const int hq = hk * group + head, t = tile * QT;
        pos = {head, tile, a.q + b * a.qs.b + hq * a.qs.h + t * a.qs.t, a.dout + ((long long)b * a.Tq + t) * gstride + hq * (2 * a.d),
               a.stat + ((long long)b * a.H + hq) * STATS * a.Tp + t};
    };
    if (first < last) go_to(first / per_head, q_first + first % per_head);
    auto issue = [&](lds_ptr dst) {
        const int have = a.Tq - pos.tile * QT;
        q_copy.issue(pos.q, have, dst);
        g_copy.issue(pos.g, have, dst + TB);
        static_assert(2 * QT % 64 == 0 && 2 * QT <= 64 * NW, "whole waves copy the statistics");
        if (wave * 64 < 2 * QT) {
            const __amdgpu_buffer_rsrc_t rs =
                __builtin_amdgcn_make_buffer_rsrc((void*)pos.stat, 0, (unsigned)((STATS - 2) * a.Tp + QT) * 4u, 0x00020000);
            const int piece = wave * 64 + lane;
            copy_piece(rs, dst + 2 * TB + wave * 1024, piece / (QT / 4) * a.Tp * 4 + piece % (QT / 4) * 16, 0);
        }
        if (pos.tile + 1 == q_tiles) {
            go_to(pos.head + 1, q_first);       // (behind the last head nothing is read any more)
        } else {
            ++pos.tile;
            pos.q += QT * a.qs.t;
            pos.g += QT * gstride;
            pos.stat += QT;
        }
    };
    // `cur` holds the tile of (head, tile), the next one goes to `fill`
    int head = pos.head, tile = pos.tile;
    Frag<T> kf[2][KS];
    const typename L::Lane rl = L::row_lane(lane), cl = L::col_lane(lane);
    // the lane's addresses, as values that the compiler cannot prove equal to those of the last use and keep
    auto fresh = [](typename L::Lane l, int off) {
        asm volatile("" : "+v"(l.mix), "+s"(off));
        return typename L::Lane{l.part + off, l.mix};
    };
    auto step = [&](bool more, lds_cptr __restrict__ cur, lds_ptr __restrict__ fill) {
        const int t0 = tile * QT + rows0, hq = hk * group + head;
        if (++tile == q_tiles) { tile = q_first; ++head; }
        if (more) issue(fill);
        if (w_first >= kend || (a.causal && t0 + 31 + reach < w_first)) return;     // nothing of this wave is seen
        const float lam = lam_of(a.lam, a.lam_bf16, hq);
        lds_cptr const gt = cur + TB;
        const SF_LDS float* const stat = (const SF_LDS float*)(cur + 2 * TB) + rows0;            // [STATS - 1][QT]
        const bool edge = w_first + 32 > kend || (a.causal && t0 < w_tmax);
        const bool wide = __any(!(fmaxf(fabsf(stat[lane & 31]), fabsf(stat[2 * QT + (lane & 31)])) < NEAR));
        const SF_LDS float* const lse = wide ? stat + 5 * QT : stat;            // or lg, with ref to be taken off the scores first
        f32x16 dp;                      // dP - delta_1
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const f32x4 dl = *(const SF_LDS f32x4*)(stat + QT + acc_row(r, h2));
#pragma unroll
            for (int e = 0; e < 4; ++e) dp[r + e] = dl[e];
        }
        const typename L::Lane gl = fresh(rl, L::row_off(rows0)), vl = fresh(rl, L::row_off(kw));
#pragma unroll
        for (int n = 0; n < VS; ++n) {
            if (n && n % 4 == 0) __builtin_amdgcn_sched_barrier(0);
            dp = mma(L::row_piece(gt, gl, 0, n), L::row_piece(vmem, vl, 0, n), dp);
        }
        f32x16 p = zero16();            // P_1 - lam P_2
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            __builtin_amdgcn_sched_barrier(0);          // (one map after the other: fewer operands in flight)
            f32x16 s = zero16();
            const typename L::Lane ql = fresh(rl, L::row_off(rows0));
#pragma unroll
            for (int n = 0; n < KS; ++n) s = mma(L::row_piece(cur, ql, 0, i * KS + n), kf[i][n], s);
            if (edge | wide) {              // (one branch: the usual tile takes none)
                if (edge) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = t0 + acc_row(r, h2) >= t_min ? s[r] : -INFINITY;
                }
                if (wide) {
#pragma unroll
                    for (int r = 0; r < 16; r += 4) {
                        const f32x4 ref = *(const SF_LDS f32x4*)(stat + (4 + 2 * i) * QT + acc_row(r, h2));
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[r + e] -= ref[e];
                    }
                }
            }
            Frag<T> df[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float ds[8];
#pragma unroll
                for (int k = 0; k < 8; k += 4) {
                    const int r = 8 * u + k;
                    const f32x4 lv = *(const SF_LDS f32x4*)(lse + 2 * QT * i + acc_row(r, h2));
                    f32x4 apart{};
                    if (i) apart = *(const SF_LDS f32x4*)(stat + 3 * QT + acc_row(r, h2));
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float y = __builtin_amdgcn_exp2f(fmaf(s[r + e], a.c, -lv[e]));
                        p[r + e] = i ? fmaf(-lam, y, p[r + e]) : y;
                        ds[k + e] = y * (i ? fmaf(-lam, dp[r + e], apart[e]) : dp[r + e]);
                    }
                }
                pack(df[u], ds);
            }
            const typename L::Lane qc = fresh(cl, L::row_off(rows0));
#pragma unroll
            for (int n = 0; n < NA / 2; ++n)
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    dk[i * (NA / 2) + n] = mma(L::col_piece(cur, qc, 16 * u, DP == 16 ? 0 : i * (NA / 2) + n), df[u], dk[i * (NA / 2) + n]);
        }
        Frag<T> pf[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = p[8 * u + j];
            pack(pf[u], x);
        }
        const typename L::Lane gc = fresh(cl, L::row_off(rows0));
#pragma unroll
        for (int n = 0; n < DT; ++n)
#pragma unroll
            for (int u = 0; u < 2; ++u) dv[n] = mma(L::col_piece(gt, gc, 16 * u, n), pf[u], dv[n]);
    };
    if (first < last) {
        const Copy<T, DP, KB, NW> vc(a.vs.t, a.d);
        vc.issue(vbase + k0 * a.vs.t, kend - k0, vmem);
        issue(buf0);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int s = 0; s < KS; ++s)
                kf[i][s] = global_piece<T>(kbase + (key < kend ? (long long)key * a.ks.t : 0), i, s * 16 + 8 * h2, a.d, key < kend);
        for (int i = first;;) {
            stage_sync();
            step(i + 1 < last, buf0, buf1);
            if (++i >= last) break;
            stage_sync();
            step(i + 1 < last, buf1, buf0);
            if (++i >= last) break;
        }
    }
    if constexpr (SPLIT) {
        join_waves<NW>(dv, (float*)smem, wave, lane);
        join_waves<NW>(dk, (float*)smem, wave, lane);
        if (wave != 0) return;
    }
    if (key >= a.Tk) return;
    const long long out = (((long long)b * a.Tk + key) * a.Hk + hk) * (2 * a.d);
    float* const po = a.part + (((long long)w.tail * w.parts + w.part) * KB + (key - k0)) * (4 * DP);
#pragma unroll
    for (int n = 0; n < DT; ++n)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int col = 32 * n + acc_row(r, h2);
            if (w.parts > 1) *reinterpret_cast<float4*>(po + col) = float4{dv[n][r], dv[n][r + 1], dv[n][r + 2], dv[n][r + 3]};
            else store_cols<T, DP>(a.dv + out, col, a.d, dv[n][r], dv[n][r + 1], dv[n][r + 2], dv[n][r + 3]);
        }
#pragma unroll
    for (int n = 0; n < NA; ++n)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int col = (DP == 16 ? 0 : 32 * n) + acc_row(r, h2), map = DP == 16 ? n : 32 * n / DP;
            if (col / DP != map) continue;
            const float4 y{dk[n][r] * a.scale, dk[n][r + 1] * a.scale, dk[n][r + 2] * a.scale, dk[n][r + 3] * a.scale};
            if (w.parts > 1) *reinterpret_cast<float4*>(po + 2 * DP + col) = y;
            else store_cols<T, DP>(a.dk + out, col, a.d, y.x, y.y, y.z, y.w);
        }
}

// adds the parts of the gradient items that were cut, in order: one wave per row (KEYS false: dq) or key (KEYS true: dv and dk)
template <typename T, int DP, bool KEYS> __global__ __launch_bounds__(256) void attn_join_grad_kernel(Args<T> a, int items, int RB) {
    constexpr int W = KEYS ? 4 * DP : 2 * DP;
    const int lane = threadIdx.x & 63, group = a.H / a.Hk;
    const long long rows = KEYS ? a.Tk : (long long)group * a.Tq, id = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int tail = (int)(id / RB), tiles = (int)((rows + RB - 1) / RB);
    if (tail >= items) return;
    int bh, x;
    locate(a.full + tail, a.B * a.Hk, tiles, a.causal, bh, x);
    const long long row = (long long)(KEYS ? x : tiles - 1 - x) * RB + id % RB;
    if (row >= rows) return;
    const int b = bh / a.Hk, hk = bh % a.Hk;
    const long long out = KEYS ? (((long long)b * a.Tk + row) * a.Hk + hk) * (2 * a.d)
                               : (((long long)b * a.Tq + row / group) * a.H + hk * group + row % group) * (2 * a.d);
    const float* const p = a.part + ((long long)tail * a.parts * RB + id % RB) * W;
    if (!KEYS && sizeof(T) == 2) {          // (there are at most 64 parts)
        const float* const sums = a.part + (long long)items * a.parts * RB * W + (long long)tail * a.parts * RB + id % RB;
        const float sum = wave_sum(lane < a.parts ? sums[(long long)lane * RB] : 0.f);
        float* const stat = a.stat + ((long long)b * a.H + hk * group + row % group) * STATS * a.Tp + row / group;
        if (lane == 0) stat[(STATS - 1LL) * a.Tp] = sum - stat[a.Tp];
    }
    for (int c = lane; c < W; c += 64) {
        const int half = c / DP & 1, j = c % DP;
        if (j >= a.d) continue;
        float s = 0.f;
        for (int i = 0; i < a.parts; ++i) s += p[(long long)i * RB * W + c];
        T* const to = KEYS ? (c < 2 * DP ? a.dv : a.dk) : a.dq;
        to[out + half * a.d + j] = from_f32<T>(s);
    }
}

// ------------------------------------------------------------------------------ host side
int padded_rows(const sf_diff_attn_desc* p) { return (p->Tq + 127) / 128 * 128; }
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
    // a launch has less than 2^32 threads: 256 for an item of 32 rows or keys, and the parts of the last ones
    const double rows = ((double)p->H / p->Hk * p->Tq + 31) / 32, keys = (p->Tk + 31) / 32;
    SF_REQUIRE((double)p->B * p->Hk * (rows > keys ? rows : keys) < 16e6, "%s: too many rows or keys for one call", who);
    return SF_OK;
}
int check_bwd_desc(const sf_diff_attn_desc* p, const char* who) {
    if (int rc = check_desc(p, who)) return rc;
    SF_REQUIRE((double)p->B * padded_rows(p) * p->H < (1 << 28), "%s: too many rows for one call", who);     // (16 threads for a row)
    return SF_OK;
}
int check_align(const void* const* ps, int n, const char* who) {
    for (int i = 0; i < n; ++i) SF_REQUIRE(ps[i] && (uintptr_t)ps[i] % 16 == 0, "%s: pointer %d is null or not 16-byte aligned", who, i);
    return SF_OK;
}

// How a launch's work items are cut.  The chip runs `slots` workgroups at a time; items beyond a whole number of rounds
// would leave most of it idle in the last one.  Those are cut into the number of parts for which the launch takes the
// least time, counted in quarters of a tile of 128 rows and 64 (f32: 32) keys, 0.5 to 1.5 us: `unit` for a step, `fixed` for what a
// part costs by itself, `join` for the launch that joins them (from sweeps of 22 shapes for each type and width).  The time is
// that of whole rounds of the longest item.  In f32 a round is 256 workgroups: one keeps a CU's matrix pipes busy, others on the
// same CU share them.  There narrow causal items, which have on average a `share` of the longest one's steps and come
// longest first, take the time of the longest or of all the work, whichever is more.
// Items of unequal length that fill the chip are not cut: they come longest first, the last ones are short.
struct Cut { int full, tail, parts; double cost; };
int width_of(const sf_diff_attn_desc* p) { return p->d <= 16 ? 0 : p->d <= 32 ? 1 : 2; }
Cut cut_items(const sf_diff_attn_desc* p, long long items, int slots, int steps, int unit, int fixed) {
    static const int joins[2][3] = {{48, 32, 32}, {32, 16, 16}};
    const bool f32 = p->dtype == SF_F32;
    const int join = joins[f32][width_of(p)];
    const double share = !p->causal ? 1 : p->Tq <= p->Tk ? 1 - (p->Tq - 1) / (2.0 * p->Tk) : (p->Tk + 1) / (2.0 * p->Tq);
    const bool rounds = !f32 || p->d > 32 || share >= 0.9;
    const int round = f32 ? 256 : slots;
    auto time = [&](long long n, int len) {
        const double one = (double)unit * len + fixed, all = n / 256.0 * (unit * len * share + fixed);
        return rounds ? (n + round - 1) / round * one : all > one ? all : one;
    };
    const long long full = items / slots * slots, tail = items - full;
    Cut best{(int)items, 0, 1, time(items, steps)};
    if (!tail || (full && share < 0.9)) return best;
    const double before = full ? time(full, steps) : 0;
    for (int n = 2; n <= 64 && steps / n >= 2; ++n) {
        const double cost = before + time(tail * n, (steps + n - 1) / n) + join;
        if (cost < best.cost) best = {(int)full, (int)tail, n, cost};
    }
    return best;
}
// workgroups that share a CU: what the kernels' registers (with split keys: LDS) leave room for
enum Pass { FWD, FWD_KEYS, DQ, DQ_KEYS, DKV, DKV_SPLIT };
int slots_of(const sf_diff_attn_desc* p, Pass pass) {
    static const int bf16_[6][3] = {{4, 3, 2}, {4, 2, 2}, {3, 3, 2}, {3, 2, 2}, {3, 2, 2}, {3, 2, 2}},
                     f32_[6][3] = {{4, 2, 1}, {2, 1, 1}, {3, 2, 1}, {2, 1, 1}, {3, 2, 1}, {2, 1, 1}};
    return 256 * (p->dtype == SF_F32 ? f32_ : bf16_)[pass][width_of(p)];
}
int fixed_of(const sf_diff_attn_desc* p) { return p->dtype == SF_F32 && p->d > 32 ? 8 : 4; }
// Up to 32 query rows per key/value head (single tokens) the waves of a workgroup share out the keys of a tile; beyond that the
// rows, or the keys where the items are too few for the chip: four times the items, and the parts are joined in LDS
// instead of by another launch.  (Forward, us, rows | keys: bf16 4 x 777 tokens, 4 heads on 2, causal, 2 x 16: 27 | 12, 2 x 64:
// 34 | 24; 1 x 4096, 4 heads, 2 x 64: 78 | 102; f32 2 x 32: 4 x 777: 54 | 42, 1 x 4096: 224 | 245.)
struct RowPlan { bool keys; int kt, rb; Cut cut; };
RowPlan row_plan(const sf_diff_attn_desc* p, Pass rows_pass, Pass keys_pass) {
    const long long rows = (long long)(p->H / p->Hk) * p->Tq, heads = (long long)p->B * p->Hk;
    const bool f32 = p->dtype == SF_F32;
    static const int fixed[2][3] = {{14, 14, 14}, {6, 12, 24}};
    const int kt = padded(p->d) == 64 ? 64 : 128;
    const RowPlan keys{true, kt, 32, cut_items(p, (rows + 31) / 32 * heads, slots_of(p, keys_pass), (p->Tk + kt - 1) / kt,
                                               f32 ? 4 : 2, fixed[f32][width_of(p)])};
    if (rows <= 32) return keys;
    const int rt = f32 ? 32 : 64;
    const RowPlan split{false, rt, 128, cut_items(p, (rows + 127) / 128 * heads, slots_of(p, rows_pass), (p->Tk + rt - 1) / rt, 4, fixed_of(p))};
    return keys.cut.cost < split.cut.cost ? keys : split;
}
RowPlan fwd_plan(const sf_diff_attn_desc* p) { return row_plan(p, FWD, FWD_KEYS); }
RowPlan dq_plan(const sf_diff_attn_desc* p) { return row_plan(p, DQ, DQ_KEYS); }
// The key gradients likewise: 128 keys, 32 for each wave, or 32 keys and the rows of a tile shared out.  (Backward pass, us, keys |
// split: bf16 2 x 365 tokens, 4 heads, 2 x 16: 30 | 21, 2 x 64: 44 | 36; 1 x 512, 8 heads, 2 x 32: 36 | 25; f32 8 x 300, 4 heads,
// causal, 2 x 16: 69 | 45.)
struct KeyPlan { bool split; int kb, qt; Cut cut; };
KeyPlan dkv_plan(const sf_diff_attn_desc* p) {
    const bool f32 = p->dtype == SF_F32;
    static const int fixed[2][3] = {{18, 18, 18}, {8, 14, 26}};
    const int group = p->H / p->Hk, heads = p->B * p->Hk, qt = padded(p->d) == 64 ? 64 : 128, unit = f32 ? 4 : 3;
    const KeyPlan split{true, 32, qt, cut_items(p, (long long)((p->Tk + 31) / 32) * heads, slots_of(p, DKV_SPLIT), (p->Tq + qt - 1) / qt * group,
                                                unit, fixed[f32][width_of(p)])};
    const KeyPlan keys{false, 128, 32, cut_items(p, (long long)((p->Tk + 127) / 128) * heads, slots_of(p, DKV), (p->Tq + 31) / 32 * group, unit,
                                                 fixed_of(p))};
    return split.cut.cost < keys.cut.cost ? split : keys;
}

template <typename T> Args<T> make_args(const sf_diff_attn_desc* p, const void* q, const void* k, const void* v, const void* lam,
                                        const int* lengths) {
    Args<T> a{};
    a.q = (const T*)q; a.k = (const T*)k; a.v = (const T*)v;
    a.qs = {p->q_stride[0], p->q_stride[1], p->q_stride[2]};
    a.ks = {p->k_stride[0], p->k_stride[1], p->k_stride[2]};
    a.vs = {p->v_stride[0], p->v_stride[1], p->v_stride[2]};
    a.lam = lam; a.lam_bf16 = p->lam_dtype == SF_BF16; a.lengths = lengths;
    a.B = p->B; a.Tq = p->Tq; a.Tp = padded_rows(p); a.Tk = p->Tk; a.H = p->H; a.Hk = p->Hk; a.d = p->d; a.causal = p->causal != 0;
    a.parts = 1;
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

template <typename T, int DP> int launch_fwd(Args<T> a, const RowPlan& f, hipStream_t st) {
    const int grid = f.cut.full + f.cut.tail * f.cut.parts;
    using L = Tile<T, DP>;
    a.full = f.cut.full;
    a.parts = f.cut.parts;
    if (f.keys) {
        constexpr int NW = DP == 64 ? 2 : 4, KT = 32 * NW;
        constexpr int box = (2 * (2 * DP / 32) * 16 + 4) * 64 * 4;
        constexpr int lds = 4 * L::bytes(KT) > box ? 4 * L::bytes(KT) : box;
        SF_LDS_ONCE((attn_fwd_kernel<T, DP, NW, true, KT>), lds);
        hipLaunchKernelGGL((attn_fwd_kernel<T, DP, NW, true, KT>), dim3(grid), dim3(64 * NW), lds, st, a);
    } else {
        constexpr int KT = sizeof(T) == 4 ? 32 : 64, lds = 4 * L::bytes(KT);
        SF_LDS_ONCE((attn_fwd_kernel<T, DP, 4, false, KT>), lds);
        hipLaunchKernelGGL((attn_fwd_kernel<T, DP, 4, false, KT>), dim3(grid), dim3(256), lds, st, a);
    }
    SF_LAUNCH_CHECK("sf_diff_attn_fwd");
    if (f.cut.tail) {
        hipLaunchKernelGGL((attn_join_kernel<T, DP>), dim3(f.cut.tail * f.rb / 4), dim3(256), 0, st, a, f.rb, f.cut.tail);
        SF_LAUNCH_CHECK("sf_diff_attn_fwd (join)");
    }
    return SF_OK;
}

template <typename T, int DP> int launch_bwd(Args<T> a, const RowPlan& f, const KeyPlan& g, hipStream_t st) {
    const long long n = (long long)a.B * a.Tp * a.H;
    using L = Tile<T, DP>;
    hipLaunchKernelGGL((attn_delta_kernel<T>), dim3(ceil_div(n, 16)), dim3(256), 0, st, a);
    SF_LAUNCH_CHECK("sf_diff_attn_bwd (delta)");
    const Cut& cq = f.cut;
    a.full = cq.full;
    a.parts = cq.parts;
    if (f.keys) {
        constexpr int NW = DP == 64 ? 2 : 4, KT = 32 * NW, box = (DP == 16 ? 2 : 2 * DP / 32) * 4096;
        constexpr int lds = 4 * L::bytes(KT) > box ? 4 * L::bytes(KT) : box;
        SF_LDS_ONCE((attn_dq_kernel<T, DP, NW, true, KT>), lds);
        hipLaunchKernelGGL((attn_dq_kernel<T, DP, NW, true, KT>), dim3(cq.full + cq.tail * cq.parts), dim3(64 * NW), lds, st, a);
    } else {
        constexpr int KT = sizeof(T) == 4 ? 32 : 64, lds = 4 * L::bytes(KT);
        SF_LDS_ONCE((attn_dq_kernel<T, DP, 4, false, KT>), lds);
        hipLaunchKernelGGL((attn_dq_kernel<T, DP, 4, false, KT>), dim3(cq.full + cq.tail * cq.parts), dim3(256), lds, st, a);
    }
    SF_LAUNCH_CHECK("sf_diff_attn_bwd (queries)");
    if (cq.tail) {
        hipLaunchKernelGGL((attn_join_grad_kernel<T, DP, false>), dim3(cq.tail * f.rb / 4), dim3(256), 0, st, a, cq.tail, f.rb);
        SF_LAUNCH_CHECK("sf_diff_attn_bwd (queries, join)");
    }
    const Cut& ck = g.cut;
    a.full = ck.full;
    a.parts = ck.parts;
    if (g.split) {
        constexpr int NW = DP == 64 ? 2 : 4, QT = 32 * NW, lds = L::bytes(32) + 2 * (2 * L::bytes(QT) + 32 * QT);
        static_assert(lds >= (2 * DP / 32 < 2 ? 2 : 2 * DP / 32) * 4096, "the waves' box");
        SF_LDS_ONCE((attn_dkv_kernel<T, DP, NW, true>), lds);
        hipLaunchKernelGGL((attn_dkv_kernel<T, DP, NW, true>), dim3(ck.full + ck.tail * ck.parts), dim3(64 * NW), lds, st, a);
    } else {
        constexpr int lds = L::bytes(128) + 2 * (2 * L::bytes(32) + 1024);
        SF_LDS_ONCE((attn_dkv_kernel<T, DP, 4, false>), lds);
        hipLaunchKernelGGL((attn_dkv_kernel<T, DP, 4, false>), dim3(ck.full + ck.tail * ck.parts), dim3(256), lds, st, a);
    }
    SF_LAUNCH_CHECK("sf_diff_attn_bwd (keys)");
    if (ck.tail) {
        hipLaunchKernelGGL((attn_join_grad_kernel<T, DP, true>), dim3(ck.tail * g.kb / 4), dim3(256), 0, st, a, ck.tail, g.kb);
        SF_LAUNCH_CHECK("sf_diff_attn_bwd (keys, join)");
    }
    return SF_OK;
}

template <typename T> int fwd(const sf_diff_attn_desc* p, const void* q, const void* k, const void* v, const void* lam,
                              const int* lengths, void* o, float* maps, float* sums, float* part, hipStream_t st) {
    Args<T> a = make_args<T>(p, q, k, v, lam, lengths);
    a.o = (T*)o; a.maps = maps; a.sums = sums; a.part = part;
    const RowPlan f = fwd_plan(p);
    const int dp = padded(p->d);
    return dp == 16 ? launch_fwd<T, 16>(a, f, st) : dp == 32 ? launch_fwd<T, 32>(a, f, st) : launch_fwd<T, 64>(a, f, st);
}
size_t stat_bytes(const sf_diff_attn_desc* p) { return (size_t)p->B * p->H * padded_rows(p) * STATS * sizeof(float); }
template <typename T> int bwd(const sf_diff_attn_desc* p, const void* q, const void* k, const void* v, const void* lam,
                              const int* lengths, const float* maps, const float* sums, const void* dout, void* dq, void* dk,
                              void* dv, void* dlam, char* ws, hipStream_t st) {
    Args<T> a = make_args<T>(p, q, k, v, lam, lengths);
    a.maps_in = maps; a.sums_in = sums; a.dout = (const T*)dout;
    a.stat = (float*)ws;
    a.part = (float*)(ws + stat_bytes(p));
    a.dq = (T*)dq; a.dk = (T*)dk; a.dv = (T*)dv;
    const int dp = padded(p->d);
    const RowPlan cq = dq_plan(p);
    const KeyPlan ck = dkv_plan(p);
    if (int rc = dp == 16 ? launch_bwd<T, 16>(a, cq, ck, st) : dp == 32 ? launch_bwd<T, 32>(a, cq, ck, st) : launch_bwd<T, 64>(a, cq, ck, st))
        return rc;
    if (dlam) {
        hipLaunchKernelGGL(attn_dlam_kernel, dim3(a.H), dim3(1024), 0, st, a.stat, dlam, a.lam_bf16, a.B, a.H, a.Tp);
        SF_LAUNCH_CHECK("sf_diff_attn_bwd (lam)");
    }
    return SF_OK;
}

}  // namespace

extern "C" size_t sf_diff_attn_fwd_workspace_bytes(const sf_diff_attn_desc* p) {
    if (check_desc(p, "sf_diff_attn_fwd_workspace_bytes")) return 0;
    const RowPlan f = fwd_plan(p);
    return (size_t)f.cut.tail * f.cut.parts * f.rb * (4 * padded(p->d) + 4) * sizeof(float);
}

extern "C" int sf_diff_attn_fwd(const sf_diff_attn_desc* p, const void* q, const void* k, const void* v, const void* lam,
                                const int* lengths, void* o, float* maps, float* sums, void* ws, size_t ws_bytes, void* stream) {
    if (int rc = check_desc(p, "sf_diff_attn_fwd")) return rc;
    const void* ps[] = {q, k, v, o};
    if (int rc = check_align(ps, 4, "sf_diff_attn_fwd")) return rc;
    SF_REQUIRE(lam && (!maps == !sums) && (uintptr_t)maps % 16 == 0 && (uintptr_t)sums % 16 == 0,
               "sf_diff_attn_fwd: lam is missing, or maps and sums are not both given and 16-byte aligned");
    const size_t need = sf_diff_attn_fwd_workspace_bytes(p);
    SF_REQUIRE(!need || (ws && ws_bytes >= need && (uintptr_t)ws % 16 == 0), "sf_diff_attn_fwd: workspace of %zu bytes is too small (%zu)",
               ws_bytes, need);
    return p->dtype == SF_BF16 ? fwd<bf16>(p, q, k, v, lam, lengths, o, maps, sums, (float*)ws, (hipStream_t)stream)
                               : fwd<float>(p, q, k, v, lam, lengths, o, maps, sums, (float*)ws, (hipStream_t)stream);
}

extern "C" size_t sf_diff_attn_bwd_workspace_bytes(const sf_diff_attn_desc* p) {
    if (check_bwd_desc(p, "sf_diff_attn_bwd_workspace_bytes")) return 0;
    const RowPlan f = dq_plan(p);
    const KeyPlan g = dkv_plan(p);
    const size_t q = (size_t)f.cut.tail * f.cut.parts * f.rb * (2 * padded(p->d) + 1), k = (size_t)g.cut.tail * g.cut.parts * g.kb * 4 * padded(p->d);
    return stat_bytes(p) + (q > k ? q : k) * sizeof(float);        // (one after the other in the same place)
}

extern "C" int sf_diff_attn_bwd(const sf_diff_attn_desc* p, const void* q, const void* k, const void* v, const void* lam,
                                const int* lengths, const float* maps, const float* sums, const void* dout, void* dq, void* dk,
                                void* dv, void* dlam, void* ws, size_t ws_bytes, void* stream) {
    if (int rc = check_bwd_desc(p, "sf_diff_attn_bwd")) return rc;
    const void* ps[] = {q, k, v, maps, dout, dq, dk, dv, sums};
    if (int rc = check_align(ps, 9, "sf_diff_attn_bwd")) return rc;
    const size_t need = sf_diff_attn_bwd_workspace_bytes(p);
    SF_REQUIRE(lam && ws && ws_bytes >= need && (uintptr_t)ws % 16 == 0, "sf_diff_attn_bwd: workspace of %zu bytes is too small (%zu)",
               ws_bytes, need);
    return p->dtype == SF_BF16
               ? bwd<bf16>(p, q, k, v, lam, lengths, maps, sums, dout, dq, dk, dv, dlam, (char*)ws, (hipStream_t)stream)
               : bwd<float>(p, q, k, v, lam, lengths, maps, sums, dout, dq, dk, dv, dlam, (char*)ws, (hipStream_t)stream);
}
