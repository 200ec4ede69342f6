// Attention among the nodes of each graph: softmax(scale * q k^T) v, forward and backward.
//
// Rows of a graph are consecutive; head h of q reads head h / (H / Hk) of k and v.  Arithmetic: fp32 results from the fp16 matrix
// cores.  Every operand is multiplied by a power of two per (graph, key head) that brings its longest row to a norm below 2^15,
// and split into two fp16 pieces (22 significant bits, an absolute floor 2^-39 below the largest row); a product is the three
// piece products hi*hi + hi*lo + lo*hi with fp32 accumulation.  Probabilities are formed in fp32 and split the same way after a
// multiplication by 2^8 ... 2^15, the gradient of the logits after one that the norms bound (|dP_ij| <= |do_i| |v_j|).
//
// Forward: one pass over the keys with the running maximum and sum of the softmax.  The logits are formed transposed
// (S^T = K Q^T), so a lane owns one query: the maximum and the sum are a lane's own business up to two exchanges, and the
// probabilities leave the product in the layout in which the next one (O^T = V^T P^T) takes them; V comes from LDS through the
// transposing loads.  Graphs of few rows are taken from the operands as they are, larger ones from images of the pieces that a pass
// of its own leaves.  Kept for the backward pass: the output and two numbers per row and head (the exponent that is subtracted and the
// inverse of the sum that is left; +inf and 0 for a row without keys).  Backward: probabilities are recomputed, once by key tiles
// (dk, dv) and once by query tiles (dq): no atomics, the same bits every time.  A query with one key has the probability 1 whatever its
// logit is: dq and dk are then zero by definition, which two roundings of dP and of its mean would not give.  A masked key's rows of k and v are taken as zeros, whatever they hold.
#include "common.h"

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int TQ = 0, TK = 1, TV = 2, TG = 3;                   // tensors: q, k, v, gradient of the output
constexpr int NO_EXP = -(1 << 20);                              // "no finite non-zero row"

struct AtArgs {
    const float* src[4]; int64_t row_stride[4], head_stride[4];     // q, k, v, do
    int64_t N; int H, Hk, R, D;
    float scale;
    const uint8_t* mask;                                        // [N] keys that take part, or null
    const int32_t* ptr;
    const int4* tiles;                                          // tiles of 64 rows: (graph, row, first tile, tiles of the graph)
    int n_tiles;
    const int4* blocks;                                         // of a launch: tiles of 64 or 128 rows, largest graphs first
    const int4* block_list[2]; int n_blocks[2];                 // all of them: (graph, row, -, -) of 64 rows, of 128 rows
    float neg;                                                  // -1, unknown to the compiler: keeps x - (float)half one instruction (v_fma_mix_f32)

    int max_rows;                                               // of the largest graph
    bool wide_g;                                                // rows of do can be read in 16 bytes (backward pass)
    int* part;                                                  // [tile][5][Hk] exponents of the longest row;  [4]: of do where rows count 2^-lift
    int* exps;                                                  // [B][Hk][4]
    int* live;                                                  // [tile] keys that take part (backward pass)
    int2* keys;                                                 // [B] keys that take part (none, one, or 2 for more), first tile of the graph
    _Float16* img[4];                                           // [heads][N][hi DP | lo DP]
    float* out;                                                 // [N, H, D]
    float2* stats;                                              // [H, N] of a row: M + lift / 64 (see row_top), and 1 / sum_j 2^(logit_j - M)
    float* delta;                                               // [H, N] sum_d do * o over the row's sum, times 2^(13 - exponent of do)
    float* dq; float* dk; float* dv;                            // [N, H or Hk, D]
};

// ---- operands into scaled fp16 pieces ------------------------------------------------------------------------------------
// Sixteen lanes take one (row, head) vector, a lane DP / 16 neighbouring columns of it.  VEC: 8- or 16-byte loads (D = DP, strides
// and addresses that allow it).
template <int DP, bool VEC>
__device__ __forceinline__ void load_part(const float* p, int sub, int D, bool live, float v[DP / 16]) {
    constexpr int E = DP / 16;
    if (VEC) {
        if (E % 4 == 0) {
#pragma unroll
            for (int i = 0; i < E; i += 4) {
                const f32x4 t = live ? *(const f32x4*)(p + sub * E + i) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < 4; ++j) v[i + j] = t[j];
            }
        } else {
#pragma unroll
            for (int i = 0; i < E; i += 2) {
                const float2 t = live ? *(const float2*)(p + sub * E + i) : make_float2(0.f, 0.f);
                v[i] = t.x; v[i + 1] = t.y;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = live && sub * E + i < D ? p[sub * E + i] : 0.f;
    }
}

// The output's gradient is divided by the row's sum here, once: the products then run on 2^(logit - M), M whole.  (With one number per
// row, log2 of the sum, its rounding alone put 3e-7 on every probability, and 2e-7 to 4e-6 of the gradients more than this way.)
template <int E>
__device__ __forceinline__ void over_sum(const AtArgs& a, int64_t n, int h, float v[E]) {
    const float f = a.stats[(int64_t)h * a.N + n].y;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] *= f;
}

// A vector of an operand, as it is split: masked keys are zeros, the gradient is over its row's sum.
template <int DP, bool VEC>
__device__ __forceinline__ void load_vec(const AtArgs& a, int ten, int64_t n, int h, float v[DP / 16]) {
    const bool masked = a.mask && (ten == TK || ten == TV);
    load_part<DP, VEC>(a.src[ten] + n * a.row_stride[ten] + h * a.head_stride[ten], threadIdx.x & 15, a.D, !(masked && !a.mask[n]), v);
    if (ten == TG) over_sum<DP / 16>(a, n, h, v);
}

// e with |row| < 2^e, from the square of the norm
__device__ __forceinline__ int above_norm(double square) { return ((((int)(__double_as_longlong(square) >> 52) & 2047) - 1023) >> 1) + 1; }

// A row keeps a whole M with sum_j 2^(logit_j - M) in [1, 2), and beside it, as 64ths, by how many powers of two its probabilities may be
// raised and stay below 2 (none where M needs the bits): the split of the logits' gradient has an absolute floor, and behind
// probabilities of 1 / n it would be met by every term.
__device__ __forceinline__ float with_lift(float M, float top) {
    return fabsf(M) < 131072.f ? fmaf(fminf(fmaxf(floorf(M - top), 0.f), 31.f), 0.015625f, M) : M;
}
__device__ __forceinline__ float row_top(float x) { return floorf(x); }
__device__ __forceinline__ int row_lift(float x) { return x < 1e30f ? (int)((x - floorf(x)) * 64.f) : 0; }

// The largest of the workgroup's values.  red: four ints of LDS.
__device__ __forceinline__ int max_of_all(int v, int* red) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v = max(v, __shfl_xor(v, o, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return max(max(red[0], red[1]), max(red[2], red[3]));
}

// One workgroup per (tile, tensor, key head) leaves the exponent e with |row| < 2^e of the tile's longest row (NO_EXP: none that is
// finite and not zero).
template <int DP, bool VEC>
__global__ __launch_bounds__(256) void k_at_norms(const AtArgs a, const int first) {
    __shared__ int red[2][4];
    const int ten = first + blockIdx.y, hk = blockIdx.z;
    const int4 tile = a.tiles[blockIdx.x];
    const int rows = min(64, (int)(a.ptr[tile.x + 1] - tile.y)), per = (ten == TQ || ten == TG) ? a.R : 1;
    int best = NO_EXP, lifted = NO_EXP;
    for (int i = threadIdx.x >> 4; i < rows * per; i += 16) {
        const int r = i / per;
        float v[DP / 16];
        load_vec<DP, VEC>(a, ten, tile.y + r, hk * per + i - r * per, v);
        double s = 0.0;
#pragma unroll
        for (int e = 0; e < DP / 16; ++e) s = fma((double)v[e], (double)v[e], s);
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) s += __shfl_xor(s, o, 64);
        if (s > 0.0 && s < 1e300) {                             // rows that hold an infinity or NaN do not count
            const int e = above_norm(s);
            best = max(best, e);
            if (ten == TG) lifted = max(lifted, e - row_lift(a.stats[(int64_t)(hk * per + i - r * per) * a.N + tile.y + r].x));
        }
    }
    best = max_of_all(best, red[0]);
    if (ten == TG) lifted = max_of_all(lifted, red[1]);
    if (threadIdx.x == 0) {
        int* p = a.part + (int64_t)blockIdx.x * 5 * a.Hk + hk;
        p[ten * a.Hk] = best;
        if (ten == TG) p[4 * a.Hk] = lifted;
    }
    if (a.live && ten == TK && hk == 0 && threadIdx.x < 64) {   // the first wave, whole
        const int i = threadIdx.x;
        const uint64_t takes = __ballot(i < rows && (!a.mask || a.mask[tile.y + i]));
        if (i == 0) a.live[blockIdx.x] = __popcll(takes);
    }
}

// One workgroup per (tile, tensor, key head) splits its rows with the exponent of the graph.  The gradient's also takes the dot products
// with the output.  Bound by memory: 32 graphs of about 5 000 nodes, four heads of 64: exponents 95 us (5.2 TB/s), pieces 168 (5.8).
// (Small graphs without the first launch, every workgroup looking through its whole graph, or one workgroup per graph that keeps it in
// registers: 32 x 138 nodes with the gradient 25 us, in two launches 19; 2 000 x 250 nodes 2.1 and 3.1 ms, in two launches 1.4.)
template <int DP, bool VEC>
__global__ __launch_bounds__(256) void k_at_split(const AtArgs a, const int first) {
    constexpr int E = DP / 16;
    __shared__ int red[4];
    const int ten = first + blockIdx.y, hk = blockIdx.z;
    const int4 tile = a.tiles[blockIdx.x];
    int e = NO_EXP;
    for (int i = threadIdx.x; i < tile.w; i += 256) e = max(e, a.part[((int64_t)(tile.z + i) * 5 + ten) * a.Hk + hk]);
    e = max_of_all(e, red);
    if (e == NO_EXP) e = 0;
    if (threadIdx.x == 0 && (int)blockIdx.x == tile.z) a.exps[((int64_t)tile.x * a.Hk + hk) * 4 + ten] = e;
    if (a.live && ten == TK && hk == 0 && (int)blockIdx.x == tile.z) {                  // the same for the whole workgroup
        int tiles = 0, most = 0;                                // that hold keys, and the keys of one of them
        for (int i = threadIdx.x; i < tile.w; i += 256) {
            const int n = a.live[tile.z + i];
            tiles += n > 0; most = max(most, n);
        }
        const bool many = __syncthreads_or(tiles > 1 || most > 1);
        const int holders = __syncthreads_count(tiles > 0);     // with not many: threads that saw one tile with one key
        if (threadIdx.x == 0) a.keys[tile.x] = make_int2(many ? 2 : min(holders, 2), tile.z);
    }
    const int rows = min(64, (int)(a.ptr[tile.x + 1] - tile.y));
    const int per = (ten == TQ || ten == TG) ? a.R : 1, sub = threadIdx.x & 15;
    for (int i = threadIdx.x >> 4; i < rows * per; i += 16) {
        const int r = i / per, h = hk * per + i - r * per;
        const int64_t n = tile.y + r;
        float v[E];
        load_vec<DP, VEC>(a, ten, n, h, v);
        f16x2 hi[E / 2], lo[E / 2];
#pragma unroll
        for (int j = 0; j < E; ++j) v[j] = ldexpf(v[j], 15 - e);
#pragma unroll
        for (int j = 0; j < E; j += 2) {
            hi[j / 2] = f16x2{(_Float16)v[j], (_Float16)v[j + 1]};
            lo[j / 2] = f16x2{(_Float16)(v[j] - (float)hi[j / 2][0]), (_Float16)(v[j + 1] - (float)hi[j / 2][1])};
        }
        _Float16* dst = a.img[ten] + ((int64_t)h * a.N + n) * (2 * DP) + sub * E;
#pragma unroll
        for (int j = 0; j < E / 2; ++j) {
            *(f16x2*)(dst + 2 * j) = hi[j];
            *(f16x2*)(dst + DP + 2 * j) = lo[j];
        }
        if (ten == TG) {
            const float* o = a.out + (n * a.H + h) * a.D;
            float dot = 0.f;
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (sub * E + j < a.D) dot = fmaf(v[j], o[sub * E + j], dot);
#pragma unroll
            for (int w = 1; w < 16; w <<= 1) dot += __shfl_xor(dot, w, 64);
            if (sub == 0) a.delta[(int64_t)h * a.N + n] = ldexpf(dot, -2);
        }
    }
}

// ---- pieces shared by the three products -----------------------------------------------------------------------------------
// Products run on v_mfma_f32_16x16x32_f16 (with real operands it delivers 1.9 PFLOP/s on this card, the 32x32x16 form 1.5: power, not
// issue, is what limits them): a row operand has lane l hold row l & 15, columns 8 (l >> 4) .. + 7 of a 32-wide slice; a column
// operand the same with columns for rows; the result has lane l hold column l & 15, rows 4 (l >> 4) + 0..3.
//
// LDS tile: a line is [hi DP | lo DP] fp16 + 16 bytes, and of 16 rows the first eight take the even lines: then neither 16 rows of
// one 16-byte chunk (row operands) nor 8 rows of two chunks (transposing loads, 32 lanes at a time) meet in one of the 64 banks.
template <int DP> constexpr int line_bytes() { return 4 * DP + 16; }
__device__ __forceinline__ int line_of(int row) { return (row & ~15) | ((row & 7) << 1) | ((row >> 3) & 1); }

// A thread's share of a tile of 64 rows on its way to LDS (threads: NT); rows from `rows` on are zeros.
template <int DP, int NT>
struct Stage {
    static constexpr int CH = 64 * (DP / 4) / NT;               // 16-byte chunks per thread
    uint4 v[CH];
    __device__ __forceinline__ void load(const _Float16* tile, int rows) {          // tile: first row in the image
        const uint4* p = (const uint4*)tile;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int f = threadIdx.x + NT * i, r = f / (DP / 4);
            v[i] = r < rows ? p[f] : make_uint4(0, 0, 0, 0);
        }
    }
    __device__ __forceinline__ void store(unsigned char* lds) const {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int f = threadIdx.x + NT * i, r = f / (DP / 4), c = f - r * (DP / 4);
            *(uint4*)(lds + line_of(r) * line_bytes<DP>() + c * 16) = v[i];
        }
    }
};

struct Frag { f16x8 hi, lo; };

// rows r0 + (lane & 15) (r0 a multiple of 16), columns 32 c + 8 (lane >> 4) ..
template <int DP>
__device__ __forceinline__ Frag row_frag(const unsigned char* lds, int r0, int c, int lane) {
    const unsigned char* p = lds + line_of(lane & 15) * line_bytes<DP>() + (lane >> 4) * 16 + r0 * line_bytes<DP>() + c * 64;
    Frag f;
    f.hi = *(const f16x8*)p;
    f.lo = *(const f16x8*)(p + 2 * DP);
    return f;
}

__device__ __forceinline__ s16x4 tr_read(const unsigned char* p) {
    typedef __attribute__((address_space(3))) s16x4 lds_v;
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v*)p);
}
// the transposed tile as a row operand: row d = 16 db + (lane & 15); its eight values are tile rows r0 + 4 g + 0..3 and
// r0 + 16 + 4 g + 0..3 (g = lane >> 4): the rows that a lane holds of two results, in the order of split_frag
template <int DP>
__device__ __forceinline__ Frag col_frag(const unsigned char* lds, int r0, int db, int lane) {
    const int i = lane & 15;
    const unsigned char* hi = lds + line_of(4 * (lane >> 4) + (i >> 2)) * line_bytes<DP>() + (i & 3) * 8 + r0 * line_bytes<DP>() + db * 32;
    const unsigned char* lo = hi + 2 * DP;
    union { struct { s16x4 a, b; } s; f16x8 v; } u, w;
    u.s.a = tr_read(hi);
    u.s.b = tr_read(hi + 16 * line_bytes<DP>());
    w.s.a = tr_read(lo);
    w.s.b = tr_read(lo + 16 * line_bytes<DP>());
    Frag f;
    f.hi = u.v; f.lo = w.v;
    return f;
}

// Two pieces of values in registers.  The large piece is cut (v_cvt_pkrtz, two values at once) rather than rounded: what is
// left then goes into the small piece whatever happened to x before.  (A plain conversion may be merged with the multiplication
// in front of it, which rounds once instead of twice, and the difference was then taken from the other result: one value in some
// thousands lost its small piece.)  The small piece is rounded to nearest: 2^-22 of x, without a drift.
__device__ __forceinline__ void split2(float x, float y, f16x2& hi, f16x2& lo, float neg) {
    union { __fp16 __attribute__((ext_vector_type(2))) a; f16x2 b; } u;
    u.a = __builtin_amdgcn_cvt_pkrtz(x, y);
    hi = u.b;
    const float rx = fmaf((float)hi[0], neg, x), ry = fmaf((float)hi[1], neg, y);
    lo = f16x2{(_Float16)rx, (_Float16)ry};
}

// ... both rounded to nearest: 2^-24.  For values that do not come out of a multiplication (v_ldexp_f32, v_exp_f32).
__device__ __forceinline__ void split2_rn(float x, float y, f16x2& hi, f16x2& lo, float neg) {
    hi = f16x2{(_Float16)x, (_Float16)y};
    lo = f16x2{(_Float16)fmaf((float)hi[0], neg, x), (_Float16)fmaf((float)hi[1], neg, y)};
}

template <bool RN = false>
__device__ __forceinline__ Frag split_frag(const f32x4& x, const f32x4& y, float neg) {
    union { Frag f; struct { f16x2 hi[4], lo[4]; } p; } u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float v0 = i < 2 ? x[2 * i] : y[2 * i - 4], v1 = i < 2 ? x[2 * i + 1] : y[2 * i - 3];
        if (RN) split2_rn(v0, v1, u.p.hi[i], u.p.lo[i], neg);
        else split2(v0, v1, u.p.hi[i], u.p.lo[i], neg);
    }
    return u.f;
}

__device__ __forceinline__ f32x4 mma3(const Frag& a, const Frag& b, f32x4 c) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.hi, b.lo, c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.lo, b.hi, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.hi, b.hi, c, 0, 0, 0);
}

// fragment of a wave's own rows, straight from the image: column operand, column = row n + (lane & 15)
template <int DP>
__device__ __forceinline__ Frag own_frag(const _Float16* img, int64_t row, int c, int lane) {
    const _Float16* p = img + row * (2 * DP) + c * 32 + (lane >> 4) * 8;
    Frag f;
    f.hi = *(const f16x8*)p;
    f.lo = *(const f16x8*)(p + DP);
    return f;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ float fold_scale(float scale, int e) {           // scale * log2(e) * 2^e
    // never zero: a zero would turn a masked logit (-inf) into NaN, and products this small are zeros either way
    return fmaxf((float)ldexp((double)scale * 1.4426950408889634, e), 1.2e-38f);
}

__device__ __forceinline__ float* row_out(float* base, int64_t n, int heads, int h, int D) { return base + (n * heads + h) * D; }

// four consecutive columns d .. d + 3 of an output row
__device__ __forceinline__ void store4(float* p, int d, int D, f32x4 v) {
    if (d + 3 < D && (D & 3) == 0) *(f32x4*)(p + d) = v;
    else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (d + i < D) p[d + i] = v[i];
    }
}

// Long sums in two steps: what the matrix cores have added over PART tiles of 64 rows goes to a second sum in LDS.  One sum alone is rounded
// six times per tile at its own size, and what out is off by enters all terms of a row of dq.  13 000 nodes, two key heads of 4, values and
// gradients with a mean, from 64 bits with one sum / two: out 1.5e-6 / 1.7e-7, dq 4.1e-5 / 3.9e-6, dk 4.7e-6 / 2.6e-7, dv 4.9e-6 / 1.8e-7;  no
// difference in time (second sums in the output's rows instead: 5 to 12 % of the kernels').  Kept where the workgroups that share a compute
// unit still fit into its LDS: everywhere but for dv of 64- and 128-wide heads and out of 96-wide ones in blocks of 128 rows.  A thread
// has SLOTS values of four columns there, `held` once there is something in them.
constexpr int PART = 16;
constexpr bool two_fit(int DP, int slots, int NW, int waves) {      // waves per SIMD that are to stay
    return (waves * 4 / NW) * (2 * 64 * (4 * DP + 16) + slots * NW * 1024 + 1024) <= 160 * 1024;
}
template <int SLOTS, int NW, bool TWO>
struct Second {
    static constexpr int FLOATS = TWO ? NW * SLOTS * 256 : 4;
    f32x4* lds;
    bool held;                                                  // the same for the whole workgroup
    __device__ __forceinline__ explicit Second(float* p) : lds((f32x4*)p), held(false) {}
    __device__ __forceinline__ f32x4& at(int slot) const { return lds[(threadIdx.x >> 6) * (SLOTS * 64) + (threadIdx.x & 63) + slot * 64]; }
    __device__ __forceinline__ void take(int slot, f32x4& v) const {                // v joins the second sum and starts again
        at(slot) = held ? at(slot) + v : v;
        v = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ void scale(int first, int step, float f) const {
        if (TWO && held) {
#pragma unroll 1
            for (int slot = first; slot < SLOTS; slot += step) at(slot) *= f;
        }
    }
    __device__ __forceinline__ f32x4 total(int slot, f32x4 v) const { return TWO && held ? at(slot) + v : v; }
};

constexpr float P_BITS = 8.f;                                   // probabilities start at 2^8 and may grow to 2^15 before a rescale
constexpr float P_GROW = 7.f;

// Waves per SIMD the registers are cut to: two (128-wide heads with 16 rows per wave and four waves: one, anything else spills).
constexpr int at_bounds(int DP, int NW) { return DP == 128 && NW == 4 ? 1 : 2; }

// ---- forward -----------------------------------------------------------------------------------------------------------------
// One tile of 64 keys (pieces in LDS) against a wave's queries.  c: what a product of the pieces is multiplied by, base 2.  RN: the
// probabilities' pieces to nearest, which shows in the sums over a few keys (graphs of two rows: 1.0e-7 -> 6.5e-8 of the result) and
// would take 3 (64 columns) to 7 % (23) of the time of large graphs.
template <int DP, int QB, bool RN, typename S2>
__device__ __forceinline__ void fwd_tile(const unsigned char* ldsK, const unsigned char* ldsV, const float* bias, bool biased, int lane,
                                         const float (&c)[QB], const Frag (&q)[QB][DP / 32], float (&m)[QB], float (&l)[QB],
                                         f32x4 (&acc)[DP / 16][QB], float neg, const S2& second, float (&most)[QB]) {
    constexpr int KC = DP / 32, DB = DP / 16;
    const int g = lane >> 4;
    f32x4 s[4][QB];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
#pragma unroll
        for (int j = 0; j < QB; ++j) s[b][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KC; ++k) {
            const Frag f = row_frag<DP>(ldsK, 16 * b, k, lane);
#pragma unroll
            for (int j = 0; j < QB; ++j) s[b][j] = mma3(f, q[j][k], s[b][j]);
        }
        if (biased) {
            const f32x4 o = *(const f32x4*)(bias + 16 * b + 4 * g);
#pragma unroll
            for (int j = 0; j < QB; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[b][j][i] = o[i] < 0.f ? -INFINITY : s[b][j][i];        // a sum would keep a NaN
        }
    }
#pragma unroll
    for (int b = 0; b < QB; ++b) {
        float top = s[0][b][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i >> 2][b][i & 3]);
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64)) * c[b];
        most[b] = fmaxf(most[b], top);
        // rescale only when a probability would leave its range
        if (__any(top > m[b] + P_GROW || (m[b] == -INFINITY && top > -INFINITY))) {
            const float mn = ceilf(fmaxf(m[b], top));      // whole: what is subtracted is then exact, and so are the rescales
            const float f = m[b] == -INFINITY ? 0.f : exp2_fast(m[b] - mn);
            m[b] = mn;
            l[b] *= f;
#pragma unroll
            for (int d = 0; d < DB; ++d) acc[d][b] *= f;
            second.scale(b, QB, f);
        }
        const float off = m[b] == -INFINITY ? 0.f : P_BITS - m[b];
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = exp2_fast(fmaf(s[i][b][j], c[b], off));
                s[i][b][j] = p;
                sum[j] += p;
            }
        l[b] += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }
#pragma unroll
    for (int kc = 0; kc < 2; ++kc) {
        Frag p[QB];
#pragma unroll
        for (int j = 0; j < QB; ++j) p[j] = split_frag<RN>(s[2 * kc][j], s[2 * kc + 1][j], neg);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            const Frag f = col_frag<DP>(ldsV, 32 * kc, d, lane);
#pragma unroll
            for (int j = 0; j < QB; ++j) acc[d][j] = mma3(f, p[j], acc[d][j]);
        }
    }
}

// The rows of a wave's queries, and their stats; ev: exponent of the values' scale.
template <int DP, int QB, typename S2>
__device__ __forceinline__ void fwd_rows(const AtArgs& a, int64_t q0, int64_t k1, int h, int lane, int ev, const float (&m)[QB], float (&l)[QB],
                                         const f32x4 (&acc)[DP / 16][QB], const S2& second, const float (&most)[QB]) {
    constexpr int DB = DP / 16;
    const int g = lane >> 4;
#pragma unroll
    for (int b = 0; b < QB; ++b) {
        l[b] += __shfl_xor(l[b], 16, 64);
        l[b] += __shfl_xor(l[b], 32, 64);
        const int64_t row = q0 + 16 * b + (lane & 15);
        if (row >= k1) continue;
        const bool none = l[b] == 0.f;
        const float f = none ? 0.f : ldexpf(1.f / l[b], ev - 15);
        float* o = row_out(a.out, row, a.H, h, a.D);
#pragma unroll
        for (int d = 0; d < DB; ++d) store4(o, 16 * d + 4 * g, a.D, none ? f32x4{0.f, 0.f, 0.f, 0.f} : second.total(d * QB + b, acc[d][b]) * f);
        if (g == 0 && a.stats) {
            const int e = (int)(__float_as_uint(l[b]) >> 23) - 127;         // l = 2^e * (1 ... 2)
            a.stats[(int64_t)h * a.N + row] = none ? make_float2(INFINITY, 0.f) : make_float2(with_lift(m[b] - P_BITS + (float)e, most[b]), ldexpf(1.f / l[b], e));
        }
    }
}

// A workgroup owns 16 * QB * NW queries of one head (a wave 16 * QB), walks the keys of the graph in tiles of 64; the next tile's loads
// are in flight during the products.  Bound by the matrix cores and the power they draw: 32 graphs of about 5 000 nodes, four heads of
// 64, 2.38 ms = 1.03 PFLOP/s of piece products, where a large fp16 product of the library reaches 1.1 (with all operands zero the three
// kernels of a training step take 8.7 instead of 10.5 ms).  Measured and not taken: waves in opposite phases of products and softmax,
// the logits of the next tile next to the softmax of this one, the 32x32x16 products, eight waves and 256 rows per workgroup,
// consecutive workgroups on one XCD (4 to 10 % slower each).
template <int DP, int QB, int NW>
__global__ __launch_bounds__(64 * NW, DP == 32 ? 4 : at_bounds(DP, NW)) void k_at_fwd(const AtArgs a) {
    constexpr int KC = DP / 32, DB = DP / 16;
    __shared__ __align__(16) unsigned char ldsK[64 * line_bytes<DP>()];
    __shared__ __align__(16) unsigned char ldsV[64 * line_bytes<DP>()];
    __shared__ __align__(16) float bias[64];
    constexpr bool TWO = two_fit(DP, DB * QB, NW, DP == 32 ? 4 : at_bounds(DP, NW));
    typedef Second<DB * QB, NW, TWO> S2;
    __shared__ __align__(16) float ldsS[S2::FLOATS];
    S2 second(ldsS);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int blk = blockIdx.x / a.H, h = blockIdx.x - blk * a.H, hk = h / a.R;
    const int4 t = a.blocks[blk];
    const int64_t k0 = a.ptr[t.x], k1 = a.ptr[t.x + 1];
    const int64_t q0 = (int64_t)t.y + 16 * QB * wave;
    const int* ex = a.exps + ((int64_t)t.x * a.Hk + hk) * 4;
    float c[QB];
#pragma unroll
    for (int b = 0; b < QB; ++b) c[b] = fold_scale(a.scale, ex[TQ] + ex[TK] - 30);
    Frag q[QB][KC];
#pragma unroll
    for (int b = 0; b < QB; ++b)
#pragma unroll
        for (int k = 0; k < KC; ++k) q[b][k] = own_frag<DP>(a.img[TQ] + (int64_t)h * a.N * (2 * DP), min(q0 + 16 * b + (lane & 15), k1 - 1), k, lane);
    f32x4 acc[DB][QB];
    float m[QB], l[QB], most[QB];                               // the exponent that is subtracted, base 2;  the sum;  the largest logit
#pragma unroll
    for (int b = 0; b < QB; ++b) { m[b] = most[b] = -INFINITY; l[b] = 0.f; }
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int b = 0; b < QB; ++b) acc[d][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    const _Float16* ki = a.img[TK] + ((int64_t)hk * a.N + k0) * (2 * DP);
    const _Float16* vi = a.img[TV] + ((int64_t)hk * a.N + k0) * (2 * DP);
    const int n = (int)(k1 - k0);
    Stage<DP, 64 * NW> sk, sv;
    sk.load(ki, min(64, n));
    sv.load(vi, min(64, n));
    float nb = threadIdx.x < 64 && (int)threadIdx.x < n && (!a.mask || a.mask[k0 + threadIdx.x]) ? 0.f : -INFINITY;
    for (int kt0 = 0; kt0 < n; kt0 += 64 * PART) {
        const int kt1 = min(n, kt0 + 64 * PART);
        for (int kt = kt0; kt < kt1; kt += 64) {
            __syncthreads();
            sk.store(ldsK);
            sv.store(ldsV);
            if (threadIdx.x < 64) bias[threadIdx.x] = nb;
            __syncthreads();
            const int next = kt + 64;
            if (next < n) {
                sk.load(ki + (int64_t)next * (2 * DP), min(64, n - next));
                sv.load(vi + (int64_t)next * (2 * DP), min(64, n - next));
                const int j = next + (int)threadIdx.x;
                nb = threadIdx.x < 64 && j < n && (!a.mask || a.mask[k0 + j]) ? 0.f : -INFINITY;
            }
            const bool biased = a.mask != nullptr || kt + 64 > n;
            fwd_tile<DP, QB, false>(ldsK, ldsV, bias, biased, lane, c, q, m, l, acc, a.neg, second, most);
        }
        if (TWO && kt1 < n) {
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int b = 0; b < QB; ++b) second.take(d * QB + b, acc[d][b]);
            second.held = true;
        }
    }
    fwd_rows<DP, QB>(a, q0, k1, h, lane, ex[TV], m, l, acc, second, most);
}

// Graphs of few rows: the operands as they are, without images.  Every workgroup splits what it multiplies on the way into the
// registers (a query's scale is its own) and into LDS (keys: a scale per tile of 64;  values: of the largest entry so far, the sums
// follow when it grows), which saves a launch and the round trip through memory.
__device__ __forceinline__ uint32_t finite_bits(float x) {      // |x| as an integer that orders like it; infinities and NaN do not count
    const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
    return u < 0x7f800000u ? u : 0u;
}
__device__ __forceinline__ int exp_above(uint32_t bits) { return max((int)(bits >> 23), 1) - 126; }      // |x| < 2^e
template <bool VEC>
__device__ __forceinline__ f32x4 four(const float* p, int d, int D, bool live) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (VEC) {
        if (live) v = *(const f32x4*)(p + d);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (live && d + i < D) v[i] = p[d + i];
    }
    return v;
}

template <int DP, int QB, int NW, bool VEC>
__global__ __launch_bounds__(64 * NW, DP == 32 ? 3 : at_bounds(DP, NW)) void k_at_fwd_small(const AtArgs a) {
    constexpr int KC = DP / 32, DB = DP / 16, NT = 64 * NW, CH = 64 * (DP / 4) / NT;
    __shared__ __align__(16) unsigned char ldsK[64 * line_bytes<DP>()];
    __shared__ __align__(16) unsigned char ldsV[64 * line_bytes<DP>()];
    __shared__ __align__(16) float bias[64];
    __shared__ uint32_t top[2][NW];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    const int blk = blockIdx.x / a.H, h = blockIdx.x - blk * a.H, hk = h / a.R;
    const int4 t = a.blocks[blk];
    const int64_t k0 = a.ptr[t.x], k1 = a.ptr[t.x + 1];
    const int64_t q0 = (int64_t)t.y + 16 * QB * wave;
    const int n = (int)(k1 - k0);
    const float* kp = a.src[TK] + hk * a.head_stride[TK];
    const float* vp = a.src[TV] + hk * a.head_stride[TV];
    f32x4 sk[CH], sv[CH];
    float nb;
    auto load = [&](int kt) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int f = threadIdx.x + NT * i, r = f / (DP / 4), d = 4 * (f - r * (DP / 4));
            const int64_t row = k0 + kt + r;
            const bool live = kt + r < n && (!a.mask || a.mask[row]);
            sk[i] = four<VEC>(kp + row * a.row_stride[TK], d, a.D, live);
            sv[i] = four<VEC>(vp + row * a.row_stride[TV], d, a.D, live);
        }
        const int j = kt + (int)threadIdx.x;
        nb = threadIdx.x < 64 && j < n && (!a.mask || a.mask[k0 + j]) ? 0.f : -INFINITY;
    };
    load(0);
    Frag q[QB][KC];
    int eq[QB];
#pragma unroll
    for (int b = 0; b < QB; ++b) {
        const float* p = a.src[TQ] + min(q0 + 16 * b + (lane & 15), k1 - 1) * a.row_stride[TQ] + h * a.head_stride[TQ];
        f32x4 x[KC][2];
        uint32_t big = 0;
#pragma unroll
        for (int k = 0; k < KC; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                x[k][i] = four<VEC>(p, 32 * k + 8 * g + 4 * i, a.D, true);
#pragma unroll
                for (int j = 0; j < 4; ++j) big = max(big, finite_bits(x[k][i][j]));
            }
        big = max(big, (uint32_t)__shfl_xor((int)big, 16, 64));
        big = max(big, (uint32_t)__shfl_xor((int)big, 32, 64));
        eq[b] = exp_above(big);
#pragma unroll
        for (int k = 0; k < KC; ++k) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) x[k][i][j] = ldexpf(x[k][i][j], 15 - eq[b]);
            q[b][k] = split_frag<true>(x[k][0], x[k][1], a.neg);
        }
    }
    f32x4 acc[DB][QB];
    float m[QB], l[QB], most[QB];
#pragma unroll
    for (int b = 0; b < QB; ++b) { m[b] = most[b] = -INFINITY; l[b] = 0.f; }
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int b = 0; b < QB; ++b) acc[d][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    const Second<1, 1, false> none(nullptr);
    int ev = -126;
    for (int kt = 0; kt < n; kt += 64) {
        uint32_t uk = 0, uv = 0;
#pragma unroll
        for (int i = 0; i < CH; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) { uk = max(uk, finite_bits(sk[i][j])); uv = max(uv, finite_bits(sv[i][j])); }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            uk = max(uk, (uint32_t)__shfl_xor((int)uk, o, 64));
            uv = max(uv, (uint32_t)__shfl_xor((int)uv, o, 64));
        }
        if (lane == 0) { top[0][wave] = uk; top[1][wave] = uv; }
        __syncthreads();                                        // also: the tile before this one has been read
#pragma unroll
        for (int w = 0; w < NW; ++w) { uk = max(uk, top[0][w]); uv = max(uv, top[1][w]); }
        const int ek = exp_above(uk), e_new = max(ev, exp_above(uv));
        if (e_new > ev) {                                       // the same for the whole workgroup
            const float f = ldexpf(1.f, ev - e_new);
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int b = 0; b < QB; ++b) acc[d][b] *= f;
            ev = e_new;
        }
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const int f = threadIdx.x + NT * i, r = f / (DP / 4), c4 = f - r * (DP / 4);
            const int off = line_of(r) * line_bytes<DP>() + c4 * 8;
            f32x4 x, y;
#pragma unroll
            for (int j = 0; j < 4; ++j) { x[j] = ldexpf(sk[i][j], 15 - ek); y[j] = ldexpf(sv[i][j], 15 - ev); }
            f16x2 hi[2], lo[2];
            split2_rn(x[0], x[1], hi[0], lo[0], a.neg);
            split2_rn(x[2], x[3], hi[1], lo[1], a.neg);
            *(f16x4*)(ldsK + off) = f16x4{hi[0][0], hi[0][1], hi[1][0], hi[1][1]};
            *(f16x4*)(ldsK + off + 2 * DP) = f16x4{lo[0][0], lo[0][1], lo[1][0], lo[1][1]};
            split2_rn(y[0], y[1], hi[0], lo[0], a.neg);
            split2_rn(y[2], y[3], hi[1], lo[1], a.neg);
            *(f16x4*)(ldsV + off) = f16x4{hi[0][0], hi[0][1], hi[1][0], hi[1][1]};
            *(f16x4*)(ldsV + off + 2 * DP) = f16x4{lo[0][0], lo[0][1], lo[1][0], lo[1][1]};
        }
        if (threadIdx.x < 64) bias[threadIdx.x] = nb;
        const bool biased = a.mask != nullptr || kt + 64 > n;
        if (kt + 64 < n) load(kt + 64);
        __syncthreads();
        float c[QB];
#pragma unroll
        for (int b = 0; b < QB; ++b) c[b] = fold_scale(a.scale, eq[b] + ek - 30);
        fwd_tile<DP, QB, true>(ldsK, ldsV, bias, biased, lane, c, q, m, l, acc, a.neg, none, most);
    }
    fwd_rows<DP, QB>(a, q0, k1, h, lane, ev, m, l, acc, none, most);
}

// ---- backward: dk and dv ---------------------------------------------------------------------------------------------------
// A workgroup owns 16 * KB * NW keys of one key head (a wave 16 * KB), walks the queries of the graph, head by head, in tiles of 64 rows.
// Two products in, two out; the same graphs 3.8 ... 4.0 ms (1.25 PFLOP/s of piece products).
template <int DP, int KB, int NW>
__global__ __launch_bounds__(64 * NW, DP == 32 ? 3 : at_bounds(DP, NW)) void k_at_dkv(const AtArgs a) {
    constexpr int KC = DP / 32, DB = DP / 16;
    __shared__ __align__(16) unsigned char ldsQ[64 * line_bytes<DP>()];
    __shared__ __align__(16) unsigned char ldsG[64 * line_bytes<DP>()];
    __shared__ __align__(16) float ldsL[64];
    __shared__ __align__(16) float ldsD[64];
    constexpr int WAVES = DP == 32 ? 3 : at_bounds(DP, NW);
    constexpr bool BOTH = two_fit(DP, 2 * DB * KB, NW, WAVES), TWO = BOTH || two_fit(DP, DB * KB, NW, WAVES);       // dk and dv, or dk alone
    typedef Second<(BOTH ? 2 : 1) * DB * KB, NW, TWO> S2;
    __shared__ __align__(16) float ldsS[S2::FLOATS];
    S2 second(ldsS);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    const int blk = blockIdx.x / a.Hk, hk = blockIdx.x - blk * a.Hk;
    const int4 t = a.blocks[blk];
    const int64_t g0 = a.ptr[t.x], g1 = a.ptr[t.x + 1];
    const int64_t key0 = (int64_t)t.y + 16 * KB * wave;
    const int* ex = a.exps + ((int64_t)t.x * a.Hk + hk) * 4;
    const float c = fold_scale(a.scale, ex[TQ] + ex[TK] - 30);
    Frag kf[KB][KC], vf[KB][KC];
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int k = 0; k < KC; ++k) {
            const int64_t row = min(key0 + 16 * b + (lane & 15), g1 - 1);
            kf[b][k] = own_frag<DP>(a.img[TK] + (int64_t)hk * a.N * (2 * DP), row, k, lane);
            vf[b][k] = own_frag<DP>(a.img[TV] + (int64_t)hk * a.N * (2 * DP), row, k, lane);
        }
    f32x4 dk[DB][KB], dv[DB][KB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int b = 0; b < KB; ++b) dk[d][b] = dv[d][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int n = (int)(g1 - g0), tiles = (n + 63) / 64, steps = tiles * a.R;
    // What the logits' gradient of a part's queries is multiplied by before it is split: 2^up, as far as their longest gradients and largest
    // probabilities allow (not the graph's).  The part's exponents are loaded one part ahead, a tile per lane.  15 200 nodes, dk from 64
    // bits with one scale / scales per part: all rows alike 7.8e-7 / 5.0e-7, one row with 1 024 times the gradient 3.8e-5 / 6.7e-7, one with
    // 1 024 times the value 7.5e-5 / 1.3e-6;  1 to 1.5 % of this kernel's time.  (A scale per tile of 64 rows: 2 to 3.5 %.)
    static_assert(TWO, "parts of dk have scales of their own");
    const int2 keys = a.keys[t.x];
    Stage<DP, 64 * NW> sq, sg;
    float nl = INFINITY, nd = 0.f;
    int up = 0;
    auto fetch = [&](int step) __attribute__((always_inline)) {
        const int hh = hk * a.R + step / tiles, r0 = (step % tiles) * 64, rows = min(64, n - r0);
        const int64_t at = (int64_t)hh * a.N + g0 + r0;
        sq.load(a.img[TQ] + at * (2 * DP), rows);
        sg.load(a.img[TG] + at * (2 * DP), rows);
        nl = INFINITY; nd = 0.f;
        if ((int)threadIdx.x < rows) {
            nl = a.stats[at + threadIdx.x].x;
            nd = a.delta[at + threadIdx.x];
        }
    };
    static_assert(PART == 16, "sixteen lanes");
    auto limits = [&](int from) __attribute__((always_inline)) {
        const int step = min(from + (lane & 15), steps - 1);
        return a.part[((int64_t)(keys.y + step % tiles) * 5 + 4) * a.Hk + hk];
    };
    int ahead = limits(0);
    fetch(0);
    for (int step0 = 0; step0 < steps; step0 += PART) {
        const int step1 = min(steps, step0 + PART);
        int top = ahead;
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) top = max(top, __shfl_xor(top, o, 64));
        up = min(__builtin_amdgcn_readfirstlane(ex[TG] - top), 60);
        if (step1 < steps) ahead = limits(step1);
        const float unit = __uint_as_float((uint32_t)(127 - 17 + up) << 23);
        for (int step = step0; step < step1; ++step) {
            __syncthreads();
            sq.store(ldsQ);
            sg.store(ldsG);
            if (threadIdx.x < 64) {
                ldsL[threadIdx.x] = -row_top(nl);
                ldsD[threadIdx.x] = ldexpf(nd, up - ex[TV]);
            }
            __syncthreads();
            if (step + 1 < steps) fetch(step + 1);
#pragma unroll
            for (int qc = 0; qc < 2; ++qc) {                        // 32 queries at a time
                Frag pf[KB], df[KB];
                {
                    f32x4 p[2][KB], s[2][KB];
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const int r0 = 32 * qc + 16 * b;
#pragma unroll
                        for (int j = 0; j < KB; ++j) p[b][j] = s[b][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int k = 0; k < KC; ++k) {
                            const Frag f = row_frag<DP>(ldsQ, r0, k, lane);
#pragma unroll
                            for (int j = 0; j < KB; ++j) p[b][j] = mma3(f, kf[j][k], p[b][j]);
                        }
#pragma unroll
                        for (int k = 0; k < KC; ++k) {
                            const Frag f = row_frag<DP>(ldsG, r0, k, lane);
#pragma unroll
                            for (int j = 0; j < KB; ++j) s[b][j] = mma3(f, vf[j][k], s[b][j]);
                        }
                        const f32x4 ls = *(const f32x4*)(ldsL + r0 + 4 * g), de = *(const f32x4*)(ldsD + r0 + 4 * g);
#pragma unroll
                        for (int j = 0; j < KB; ++j)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                p[b][j][i] = exp2_fast(fmaf(p[b][j][i], c, ls[i]));
                                s[b][j][i] = p[b][j][i] * fmaf(s[b][j][i], unit, -de[i]);
                                p[b][j][i] *= 0x1p14f;
                            }
                    }
#pragma unroll
                    for (int j = 0; j < KB; ++j) {
                        pf[j] = split_frag(p[0][j], p[1][j], a.neg);
                        df[j] = split_frag(s[0][j], s[1][j], a.neg);
                    }
                }
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const Frag f = col_frag<DP>(ldsG, 32 * qc, d, lane);
#pragma unroll
                    for (int j = 0; j < KB; ++j) dv[d][j] = mma3(f, pf[j], dv[d][j]);
                }
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const Frag f = col_frag<DP>(ldsQ, 32 * qc, d, lane);
#pragma unroll
                    for (int j = 0; j < KB; ++j) dk[d][j] = mma3(f, df[j], dk[d][j]);
                }
            }
        }
        if (TWO && step1 < steps) {
            const float down = ldexpf(1.f, -up);
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int b = 0; b < KB; ++b) {
                    dk[d][b] *= down;
                    second.take(d * KB + b, dk[d][b]);
                    if (BOTH) second.take((DB + d) * KB + b, dv[d][b]);
                }
            second.held = true;
        }
    }
#pragma unroll
    for (int b = 0; b < KB; ++b) {
        const int64_t row = key0 + 16 * b + (lane & 15);
        if (row >= g1) continue;
        const bool live = !a.mask || a.mask[row], many = keys.x > 1;
        float* pk = row_out(a.dk, row, a.Hk, hk, a.D);
        float* pv = row_out(a.dv, row, a.Hk, hk, a.D);
        const float down = ldexpf(1.f, -up);
        const int ek = ex[TG] + ex[TV] + ex[TQ] - 28, ev = ex[TG] - 29;
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            f32x4 x = second.total(d * KB + b, dk[d][b] * down), y = BOTH ? second.total((DB + d) * KB + b, dv[d][b]) : dv[d][b];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = live && many ? ldexpf(x[i] * a.scale, ek) : 0.f;
                y[i] = live ? ldexpf(y[i], ev) : 0.f;
            }
            store4(pk, 16 * d + 4 * g, a.D, x);
            store4(pv, 16 * d + 4 * g, a.D, y);
        }
    }
}

// ---- backward: dq -----------------------------------------------------------------------------------------------------------
// A workgroup owns 16 * QB * NW queries of one head and walks the keys as the forward pass does; two products in, one out; the same
// graphs 2.9 ... 3.0 ms (1.25 PFLOP/s).  One kernel for dq, dk and dv would save two of the seven products but has to add dq over key
// tiles, by atomics whose order changes results, or through memory.
//
// The incoming gradient comes from the operand itself and not from its image: each query's row has a power of two of its own, by the
// row's own norm, up to the split of the logits' gradient.  With the scale of the longest row, a row F times shorter reached that split
// log2 F bits lower, behind probabilities of 1 / n already (one row of 5 000 with 16 384 times the others' gradient, the others' dq by row:
// 1.6e-3 from 64 bits; so 8e-7, the formulas in fp32 2.5e-6).  A row's probabilities are raised by its lift on the way (one value of 15 200
// 1 024 times the others: dq 4.6e-5 without, 6.3e-7 with).
template <int DP, int QB, int NW>
__global__ __launch_bounds__(64 * NW, DP == 32 ? 3 : at_bounds(DP, NW)) void k_at_dq(const AtArgs a) {
    constexpr int KC = DP / 32, DB = DP / 16;
    __shared__ __align__(16) unsigned char ldsK[64 * line_bytes<DP>()];
    __shared__ __align__(16) unsigned char ldsV[64 * line_bytes<DP>()];
    __shared__ __align__(16) float bias[64];
    constexpr bool TWO = two_fit(DP, DB * QB, NW, DP == 32 ? 3 : at_bounds(DP, NW));
    typedef Second<DB * QB, NW, TWO> S2;
    __shared__ __align__(16) float ldsS[S2::FLOATS];
    S2 second(ldsS);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    const int blk = blockIdx.x / a.H, h = blockIdx.x - blk * a.H, hk = h / a.R;
    const int4 t = a.blocks[blk];
    const int64_t k0 = a.ptr[t.x], k1 = a.ptr[t.x + 1];
    const int64_t q0 = (int64_t)t.y + 16 * QB * wave;
    if (a.keys[t.x].x < 2) {                                      // the same for the whole workgroup
#pragma unroll
        for (int b = 0; b < QB; ++b) {
            const int64_t row = q0 + 16 * b + (lane & 15);
            if (row >= k1) continue;
#pragma unroll
            for (int d = 0; d < DB; ++d) store4(row_out(a.dq, row, a.H, h, a.D), 16 * d + 4 * g, a.D, f32x4{0.f, 0.f, 0.f, 0.f});
        }
        return;
    }
    const int* ex = a.exps + ((int64_t)t.x * a.Hk + hk) * 4;
    const float c = fold_scale(a.scale, ex[TQ] + ex[TK] - 30);
    Frag q[QB][KC], go[QB][KC];
    float ls[QB], de[QB];
    int eg[QB], lift[QB];                                       // exponent of the row's own scale
#pragma unroll
    for (int b = 0; b < QB; ++b) {
        const int64_t row = min(q0 + 16 * b + (lane & 15), k1 - 1);
        const float2 st = a.stats[(int64_t)h * a.N + row];
        const float* p = a.src[TG] + row * a.row_stride[TG] + h * a.head_stride[TG];
        f32x4 x[KC][2];
        double sum = 0.0;
#pragma unroll
        for (int k = 0; k < KC; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int d = 32 * k + 8 * g + 4 * i;
                x[k][i] = a.wide_g ? four<true>(p, d, a.D, true) : four<false>(p, d, a.D, true);
#pragma unroll
                for (int j = 0; j < 4; ++j) { x[k][i][j] *= st.y; sum = fma((double)x[k][i][j], (double)x[k][i][j], sum); }
            }
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        eg[b] = sum > 0.0 && sum < 1e300 ? above_norm(sum) : ex[TG];
#pragma unroll
        for (int k = 0; k < KC; ++k) {
            q[b][k] = own_frag<DP>(a.img[TQ] + (int64_t)h * a.N * (2 * DP), row, k, lane);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) x[k][i][j] = ldexpf(x[k][i][j], 15 - eg[b]);
            go[b][k] = split_frag<true>(x[k][0], x[k][1], a.neg);
        }
        lift[b] = row_lift(st.x);
        ls[b] = (float)lift[b] - row_top(st.x);                 // probabilities of up to 1 ... 2
        de[b] = ldexpf(a.delta[(int64_t)h * a.N + row], ex[TG] - eg[b] - ex[TV]);
    }
    f32x4 acc[DB][QB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int b = 0; b < QB; ++b) acc[d][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    const _Float16* ki = a.img[TK] + ((int64_t)hk * a.N + k0) * (2 * DP);
    const _Float16* vi = a.img[TV] + ((int64_t)hk * a.N + k0) * (2 * DP);
    const int n = (int)(k1 - k0);
    Stage<DP, 64 * NW> sk, sv;
    sk.load(ki, min(64, n));
    sv.load(vi, min(64, n));
    float nb = threadIdx.x < 64 && (int)threadIdx.x < n && (!a.mask || a.mask[k0 + threadIdx.x]) ? 0.f : -INFINITY;
    for (int kt0 = 0; kt0 < n; kt0 += 64 * PART) {
        const int kt1 = min(n, kt0 + 64 * PART);
        for (int kt = kt0; kt < kt1; kt += 64) {
            __syncthreads();
            sk.store(ldsK);
            sv.store(ldsV);
            if (threadIdx.x < 64) bias[threadIdx.x] = nb;
            __syncthreads();
            const int next = kt + 64;
            if (next < n) {
                sk.load(ki + (int64_t)next * (2 * DP), min(64, n - next));
                sv.load(vi + (int64_t)next * (2 * DP), min(64, n - next));
                const int j = next + (int)threadIdx.x;
                nb = threadIdx.x < 64 && j < n && (!a.mask || a.mask[k0 + j]) ? 0.f : -INFINITY;
            }
            const bool biased = a.mask != nullptr || kt + 64 > n;
#pragma unroll
            for (int kc = 0; kc < 2; ++kc) {
                Frag df[QB];
                {
                    f32x4 p[2][QB], s[2][QB];
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const int r0 = 32 * kc + 16 * b;
#pragma unroll
                        for (int j = 0; j < QB; ++j) p[b][j] = s[b][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int k = 0; k < KC; ++k) {
                            const Frag f = row_frag<DP>(ldsK, r0, k, lane);
#pragma unroll
                            for (int j = 0; j < QB; ++j) p[b][j] = mma3(f, q[j][k], p[b][j]);
                        }
#pragma unroll
                        for (int k = 0; k < KC; ++k) {
                            const Frag f = row_frag<DP>(ldsV, r0, k, lane);
#pragma unroll
                            for (int j = 0; j < QB; ++j) s[b][j] = mma3(f, go[j][k], s[b][j]);
                        }
                        if (biased) {
                            const f32x4 o = *(const f32x4*)(bias + r0 + 4 * g);
#pragma unroll
                            for (int j = 0; j < QB; ++j) p[b][j] += o;
                        }
#pragma unroll
                        for (int j = 0; j < QB; ++j)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float e = exp2_fast(fmaf(p[b][j][i], c, ls[j]));
                                s[b][j][i] = e * fmaf(s[b][j][i], 0x1p-17f, -de[j]);
                            }
                    }
#pragma unroll
                    for (int j = 0; j < QB; ++j) df[j] = split_frag(s[0][j], s[1][j], a.neg);
                }
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const Frag f = col_frag<DP>(ldsK, 32 * kc, d, lane);
#pragma unroll
                    for (int j = 0; j < QB; ++j) acc[d][j] = mma3(f, df[j], acc[d][j]);
                }
            }
        }
        if (TWO && kt1 < n) {
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int b = 0; b < QB; ++b) second.take(d * QB + b, acc[d][b]);
            second.held = true;
        }
    }
#pragma unroll
    for (int b = 0; b < QB; ++b) {
        const int64_t row = q0 + 16 * b + (lane & 15);
        if (row >= k1) continue;
        float* o = row_out(a.dq, row, a.H, h, a.D);
        const int e = eg[b] - lift[b] + ex[TV] + ex[TK] - 28;
#pragma unroll
        for (int d = 0; d < DB; ++d) {
            f32x4 x = second.total(d * QB + b, acc[d][b]);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = ldexpf(x[i] * a.scale, e);
            store4(o, 16 * d + 4 * g, a.D, x);
        }
    }
}

// ---- host side ----------------------------------------------------------------------------------------------------------------
int at_dp(int D) { return (D + 31) / 32 * 32; }

constexpr int SMALL_ROWS = 512;                                 // forward: no images where no graph is larger
bool at_no_images(bool backward, int max_rows) { return !backward && max_rows <= SMALL_ROWS; }

struct AtSizes { size_t part, exps, live, keys, img[4], delta, total; };
AtSizes at_sizes(int64_t N, int H, int Hk, int D, int64_t n_tiles, int64_t graphs, bool backward) {
    AtSizes s;
    const size_t row = (size_t)at_dp(D) * 4;
    s.part = hgv_align256((size_t)n_tiles * 5 * Hk * sizeof(int));
    s.exps = hgv_align256((size_t)graphs * Hk * 4 * sizeof(int));
    s.live = backward ? hgv_align256((size_t)n_tiles * sizeof(int)) : 0;
    s.keys = backward ? hgv_align256((size_t)graphs * sizeof(int2)) : 0;
    s.img[TQ] = hgv_align256((size_t)N * H * row);
    s.img[TK] = s.img[TV] = hgv_align256((size_t)N * Hk * row);
    s.img[TG] = backward ? s.img[TQ] : 0;
    s.delta = backward ? hgv_align256((size_t)N * H * sizeof(float)) : 0;
    s.total = s.part + s.exps + s.live + s.keys + s.img[0] + s.img[1] + s.img[2] + s.img[3] + s.delta;
    return s;
}

template <typename F>
void at_rows(AtArgs& a, int heads, F launch) {
    // blocks of 128 rows where that gives a workgroup to each of the 256 compute units, else of 64 (one graph of 5 000 nodes, one
    // head: forward and backward 0.47 ms)
    const int i = (int64_t)a.n_blocks[1] * heads >= 256 ? 1 : 0;
    a.blocks = a.block_list[i];
    launch(i, dim3((unsigned)((int64_t)a.n_blocks[i] * heads)));
}

// The operands' images: tensors first .. last.
template <int DP, bool VEC>
void at_images(const AtArgs& a, int first, int last, hipStream_t stream) {
    const dim3 grid((unsigned)a.n_tiles, (unsigned)(last - first + 1), (unsigned)a.Hk);
    hipLaunchKernelGGL((k_at_norms<DP, VEC>), grid, dim3(256), 0, stream, a, first);
    hipLaunchKernelGGL((k_at_split<DP, VEC>), grid, dim3(256), 0, stream, a, first);
}

template <int DP>
int at_launch(AtArgs a, bool backward, hipStream_t stream) {
    bool vec = a.D == DP;
    for (int i = 0; i < (backward ? 4 : 3); ++i)
        vec = vec && hgv_aligned(a.src[i], 16) && a.row_stride[i] % 4 == 0 && a.head_stride[i] % 4 == 0;
    a.wide_g = vec;
    // Without images where no graph is large: what splitting every operand once per workgroup costs stays below a pass of its own over
    // memory (four heads of 64, with and without: 32 graphs of 138 nodes 15 and 26 us, 2 000 of 250 0.70 and 1.74 ms, 200 of 512 0.26
    // and 0.37, 100 of 1 000 0.43 and 0.51, 16 of 5 000 1.44 and 1.29; six heads of 23: 200 of 512 0.24 and 0.26, 100 of 1 000 0.39
    // and 0.35).
    if (at_no_images(backward, a.max_rows)) {
        constexpr int QB = DP <= 64 ? 2 : 1;
        at_rows(a, a.H, [&](int i, dim3 grid) {
            if (i && vec) hipLaunchKernelGGL((k_at_fwd_small<DP, QB, 8 / QB, true>), grid, dim3(512 / QB), 0, stream, a);
            else if (i) hipLaunchKernelGGL((k_at_fwd_small<DP, QB, 8 / QB, false>), grid, dim3(512 / QB), 0, stream, a);
            else if (vec) hipLaunchKernelGGL((k_at_fwd_small<DP, 1, 4, true>), grid, dim3(256), 0, stream, a);
            else hipLaunchKernelGGL((k_at_fwd_small<DP, 1, 4, false>), grid, dim3(256), 0, stream, a);
        });
        HGV_CHECK_LAUNCH("graph_attention_fwd");
        return HGV_OK;
    }
    if (vec) at_images<DP, true>(a, TQ, backward ? TG : TV, stream);
    else at_images<DP, false>(a, TQ, backward ? TG : TV, stream);
    // 32 rows per wave, four waves; wider heads (above 64 columns backward, 96 forward): 16 rows, eight waves, so that the accumulators
    // do not push the operands out of the registers; blocks of 64 rows: 16 rows, four waves.  32 x 2 500 nodes, 64 columns, backward:
    // 32 rows 2.05 ms, 16 rows 2.25; 128 columns forward: 32 rows (with spills) 1.15 ms, 16 rows 0.79.
    constexpr int RB = DP <= 64 ? 2 : 1;
    if (!backward) {
        constexpr int QB = DP <= 96 ? 2 : 1;
        at_rows(a, a.H, [&](int i, dim3 grid) {
            if (i) hipLaunchKernelGGL((k_at_fwd<DP, QB, 8 / QB>), grid, dim3(512 / QB), 0, stream, a);
            else hipLaunchKernelGGL((k_at_fwd<DP, 1, 4>), grid, dim3(256), 0, stream, a);
        });
    } else {
        if (a.dk) at_rows(a, a.Hk, [&](int i, dim3 grid) {
            if (i) hipLaunchKernelGGL((k_at_dkv<DP, RB, 8 / RB>), grid, dim3(512 / RB), 0, stream, a);
            else hipLaunchKernelGGL((k_at_dkv<DP, 1, 4>), grid, dim3(256), 0, stream, a);
        });
        if (a.dq) at_rows(a, a.H, [&](int i, dim3 grid) {
            if (i) hipLaunchKernelGGL((k_at_dq<DP, RB, 8 / RB>), grid, dim3(512 / RB), 0, stream, a);
            else hipLaunchKernelGGL((k_at_dq<DP, 1, 4>), grid, dim3(256), 0, stream, a);
        });
    }
    HGV_CHECK_LAUNCH(backward ? "graph_attention_bwd" : "graph_attention_fwd");
    return HGV_OK;
}

int at_dispatch(const AtArgs& a, bool backward, hipStream_t stream) {
    switch (at_dp(a.D)) {
        case 32: return at_launch<32>(a, backward, stream);
        case 64: return at_launch<64>(a, backward, stream);
        case 96: return at_launch<96>(a, backward, stream);
        default: return at_launch<128>(a, backward, stream);
    }
}

int at_fill(AtArgs& a, const char* what, int64_t N, int num_graphs, int H, int Hk, int D, float scale, const uint8_t* mask, const int32_t* ptr,
            int max_rows, const int32_t* tiles, int n_tiles, const int32_t* blocks, int n64, int n128, void* ws, size_t ws_bytes, bool backward) {
    HGV_REQUIRE(N > 0 && N <= 0x7fffffff && num_graphs > 0 && H > 0 && Hk > 0 && H % Hk == 0 && D > 0, HGV_EINVAL, "%s: bad sizes", what);
    HGV_REQUIRE(D <= 128 && H <= 65535, HGV_EUNSUPPORTED, "%s: heads of %d columns (at most 128), %d of them", what, D, H);
    HGV_REQUIRE(scale > 0.f && scale < INFINITY, HGV_EINVAL, "%s: the scale must be positive and finite", what);
    HGV_REQUIRE(ptr && tiles && blocks && n_tiles > 0 && n64 > 0 && n128 > 0 && max_rows > 0, HGV_EINVAL, "%s: null plan", what);
    HGV_REQUIRE((int64_t)n64 * H <= 0x3fffffff, HGV_EUNSUPPORTED, "%s: too many tiles", what);
    const AtSizes s = at_sizes(N, H, Hk, D, n_tiles, num_graphs, backward);
    const size_t need = at_no_images(backward, max_rows) ? 256 : s.total;
    HGV_REQUIRE(ws && ws_bytes >= need && hgv_aligned(ws, 256), HGV_EWORKSPACE, "%s: workspace too small or misaligned", what);
    a.neg = -1.f;
    a.N = N; a.H = H; a.Hk = Hk; a.R = H / Hk; a.D = D; a.scale = scale; a.mask = mask; a.ptr = ptr;
    a.tiles = (const int4*)tiles; a.n_tiles = n_tiles; a.max_rows = max_rows;
    a.n_blocks[0] = n64; a.n_blocks[1] = n128;
    a.block_list[0] = (const int4*)blocks; a.block_list[1] = a.block_list[0] + n64;
    if (at_no_images(backward, max_rows)) return HGV_OK;
    char* p = (char*)ws;
    a.part = (int*)p; p += s.part;
    a.exps = (int*)p; p += s.exps;
    if (backward) {
        a.live = (int*)p; p += s.live;
        a.keys = (int2*)p; p += s.keys;
    }
    for (int i = 0; i < 4; ++i) { a.img[i] = (_Float16*)p; p += s.img[i]; }
    a.delta = (float*)p;
    return HGV_OK;
}

}  // namespace

extern "C" size_t hgv_graph_attention_ws(int64_t N, int num_graphs, int H, int Hk, int D, int64_t n_tiles, int backward) {
    if (N <= 0 || num_graphs <= 0 || H <= 0 || Hk <= 0 || D <= 0 || n_tiles <= 0) return 0;
    return at_sizes(N, H, Hk, D, n_tiles, num_graphs, backward != 0).total;
}

extern "C" size_t hgv_graph_attention_fwd_ws(int64_t N, int num_graphs, int H, int Hk, int D, int64_t n_tiles, int max_rows) {
    const size_t all = hgv_graph_attention_ws(N, num_graphs, H, Hk, D, n_tiles, 0);
    return all && at_no_images(false, max_rows) ? 256 : all;
}

extern "C" int hgv_graph_attention_fwd(const float* q, int64_t q_row, int64_t q_head, const float* k, int64_t k_row, int64_t k_head,
                                       const float* v, int64_t v_row, int64_t v_head, int64_t N, int num_graphs, int H, int Hk, int D,
                                       float scale, const uint8_t* mask, const int32_t* ptr, int max_rows, const int32_t* tiles, int n_tiles,
                                       const int32_t* blocks, int n64, int n128, float* out, float* stats, void* ws, size_t ws_bytes,
                                       hipStream_t stream) {
    AtArgs a = {};
    const int rc = at_fill(a, "graph_attention_fwd", N, num_graphs, H, Hk, D, scale, mask, ptr, max_rows, tiles, n_tiles, blocks, n64, n128, ws, ws_bytes, false);
    if (rc) return rc;
    HGV_REQUIRE(q && k && v && out && (D % 4 || hgv_aligned(out, 16)) && hgv_aligned(stats, 8), HGV_EINVAL, "graph_attention_fwd: null or misaligned buffer");
    a.src[TQ] = q; a.row_stride[TQ] = q_row; a.head_stride[TQ] = q_head;
    a.src[TK] = k; a.row_stride[TK] = k_row; a.head_stride[TK] = k_head;
    a.src[TV] = v; a.row_stride[TV] = v_row; a.head_stride[TV] = v_head;
    a.out = out; a.stats = (float2*)stats;
    return at_dispatch(a, false, stream);
}

extern "C" int hgv_graph_attention_bwd(const float* q, int64_t q_row, int64_t q_head, const float* k, int64_t k_row, int64_t k_head,
                                       const float* v, int64_t v_row, int64_t v_head, const float* g, int64_t g_row, int64_t g_head,
                                       const float* out, const float* stats, int64_t N, int num_graphs, int H, int Hk, int D, float scale,
                                       const uint8_t* mask, const int32_t* ptr, int max_rows, const int32_t* tiles, int n_tiles, const int32_t* blocks,
                                       int n64, int n128, float* dq, float* dk, float* dv, void* ws, size_t ws_bytes, hipStream_t stream) {
    AtArgs a = {};
    const int rc = at_fill(a, "graph_attention_bwd", N, num_graphs, H, Hk, D, scale, mask, ptr, max_rows, tiles, n_tiles, blocks, n64, n128, ws, ws_bytes, true);
    if (rc) return rc;
    HGV_REQUIRE(q && k && v && g && out && stats && hgv_aligned(stats, 8) && (dq || dk) && !dk == !dv, HGV_EINVAL, "graph_attention_bwd: null buffer (dk and dv come together)");
    HGV_REQUIRE(D % 4 || (hgv_aligned(dq, 16) && hgv_aligned(dk, 16) && hgv_aligned(dv, 16)), HGV_EINVAL, "graph_attention_bwd: misaligned buffer");
    a.src[TQ] = q; a.row_stride[TQ] = q_row; a.head_stride[TQ] = q_head;
    a.src[TK] = k; a.row_stride[TK] = k_row; a.head_stride[TK] = k_head;
    a.src[TV] = v; a.row_stride[TV] = v_row; a.head_stride[TV] = v_head;
    a.src[TG] = g; a.row_stride[TG] = g_row; a.head_stride[TG] = g_head;
    a.out = (float*)out; a.stats = (float2*)stats; a.dq = dq; a.dk = dk; a.dv = dv;
    return at_dispatch(a, true, stream);
}
