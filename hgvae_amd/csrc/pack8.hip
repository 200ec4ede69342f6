// Activation checkpoints in 8 bits: a row-major fp32 matrix as 8-bit integers with one power of two for each row and block
// of 32 columns, and back.
//
// For a block with largest magnitude amax:  e = floor(log2 amax) - 6, one more where amax >= 127.5 * 2^e, held in [-126, 121];
// q = round_to_nearest_even(x * 2^-e), |q| <= 127 (cut only beyond 127.5 * 2^121); the stored byte is e + 127 and the value that stands for x is q * 2^e.
// A power of two makes both products exact (so the quotient is the same in any precision), and q * 2^e has at most 7
// significant bits: it is exact in bf16 too, which is what the weight gradient reads.  |value - x| <= 2^(e-1) <= amax / 126
// for amax >= 2^-120.  A block that holds an infinity or a NaN gets the byte 255 and reads back as NaN.
#include "pack8.h"
#include <type_traits>

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// Eight lanes take one block of 32 columns of one row (a lane four columns); the 32 lane groups of a workgroup cover
// floor(32 / blocks) rows at a time (wide matrices: 32 blocks of one row, further blocks in blockIdx.y), and walk rows with
// that stride.  Bound by memory: 4 bytes read and 1.03 written per element.  160 001 x 256: 30 us, 6.9 TB/s (part of it from the
// memory-side cache); back 30 us with streaming stores, 31 with ordinary ones but 6 us more until the next launch starts.
template <bool VEC>
__global__ __launch_bounds__(256) void k_pack8(const float* __restrict__ x, int64_t ldx, int64_t N, int C, int8_t* __restrict__ q,
                                               int64_t ldq, uint8_t* __restrict__ scale, int nb, int per_pass, int rows_per_wg) {
    const int grp = threadIdx.x >> 3, sub = threadIdx.x & 7;
    const int j0 = blockIdx.y * 32, jn = min(nb - j0, 32);
    const int r = grp / jn, j = j0 + grp - r * jn;
    if (r >= per_pass) return;                                  // whole lane groups leave: the shuffles below stay inside one
    const int c = 32 * j + 4 * sub;
    const int64_t base = (int64_t)blockIdx.x * rows_per_wg;
    const int64_t end = min(base + rows_per_wg, N);
    for (int64_t n = base + r; n < end; n += per_pass) {
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        const float* p = x + n * ldx + c;
        if (VEC) {
            if (c < C) {
                const float4 t = *(const float4*)p;
                v[0] = t.x;
                v[1] = c + 1 < C ? t.y : 0.f;
                v[2] = c + 2 < C ? t.z : 0.f;
                v[3] = c + 3 < C ? t.w : 0.f;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c + i < C) v[i] = p[i];
        }
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
        const int byte = p8_byte(p8_max8(m));
        const uint32_t packed = p8_quantise4(v, byte);
        if (c < ldq) *(uint32_t*)(q + n * ldq + c) = packed;
        if (sub == 0) scale[n * nb + j] = (uint8_t)byte;
    }
}

template <bool VEC>
__global__ __launch_bounds__(256) void k_unpack8(const int8_t* __restrict__ q, int64_t ldq, const uint8_t* __restrict__ scale, int nb,
                                                 int64_t N, int C, float* __restrict__ out, int64_t ldo, int per_pass,
                                                 int rows_per_wg) {
    const int grp = threadIdx.x >> 3, sub = threadIdx.x & 7;
    const int j0 = blockIdx.y * 32, jn = min(nb - j0, 32);
    const int r = grp / jn, j = j0 + grp - r * jn;
    const int c = 32 * j + 4 * sub;
    if (r >= per_pass || c >= C) return;
    const int64_t base = (int64_t)blockIdx.x * rows_per_wg;
    const int64_t end = min(base + rows_per_wg, N);
    for (int64_t n = base + r; n < end; n += per_pass) {
        const uint32_t w = *(const uint32_t*)(q + n * ldq + c);
        float v[4];
        p8_values4(w, scale[n * nb + j], v);
        float* p = out + n * ldo + c;
        if (VEC) __builtin_nontemporal_store(f32x4{v[0], v[1], v[2], v[3]}, (f32x4*)p);      // bytes behind the last column are zero
        else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (c + i < C) p[i] = v[i];
        }
    }
}

struct P8Grid { dim3 grid; int per_pass, rows; };
P8Grid p8_grid(int64_t N, int nb) {
    P8Grid g;
    g.per_pass = nb >= 32 ? 1 : 32 / nb;
    // eight passes of a workgroup where that still leaves a few thousand workgroups
    const int slabs = (nb + 31) / 32;
    int passes = 8;
    while (passes > 1 && hgv_cdiv(N, (int64_t)g.per_pass * passes) * slabs < 4096) passes >>= 1;
    while (hgv_cdiv(N, (int64_t)g.per_pass * passes) > 0x7fffffff) passes *= 2;
    g.rows = g.per_pass * passes;
    g.grid = dim3((unsigned)hgv_cdiv(N, g.rows), (unsigned)slabs);
    return g;
}

}  // namespace

extern "C" int hgv_pack8(const float* x, int64_t ldx, int64_t N, int C, int8_t* q, int64_t ldq, uint8_t* scale, hipStream_t stream) {
    HGV_REQUIRE(N >= 0 && C > 0, HGV_EINVAL, "pack8: bad sizes");
    if (N == 0) return HGV_OK;
    HGV_REQUIRE(x && q && scale && ldx >= C && ldq >= C && ldq % 16 == 0 && hgv_aligned(q, 16), HGV_EINVAL,
                "pack8: null / misaligned buffer or bad leading dimension");
    const int nb = (C + 31) / 32;
    HGV_REQUIRE(ldq <= 32 * (int64_t)nb, HGV_EINVAL, "pack8: the leading dimension of q reaches behind its last block");
    HGV_REQUIRE(nb <= 32 * 65535, HGV_EUNSUPPORTED, "pack8: too many columns");
    const P8Grid g = p8_grid(N, nb);
    const bool vec = hgv_aligned(x, 16) && ldx % 4 == 0 && ldx >= (C + 3) / 4 * 4;
    if (vec) hipLaunchKernelGGL(k_pack8<true>, g.grid, dim3(256), 0, stream, x, ldx, N, C, q, ldq, scale, nb, g.per_pass, g.rows);
    else hipLaunchKernelGGL(k_pack8<false>, g.grid, dim3(256), 0, stream, x, ldx, N, C, q, ldq, scale, nb, g.per_pass, g.rows);
    HGV_CHECK_LAUNCH("pack8");
    return HGV_OK;
}

extern "C" int hgv_unpack8(const int8_t* q, int64_t ldq, const uint8_t* scale, int64_t N, int C, float* out, int64_t ldo,
                           hipStream_t stream) {
    HGV_REQUIRE(N >= 0 && C > 0, HGV_EINVAL, "unpack8: bad sizes");
    if (N == 0) return HGV_OK;
    HGV_REQUIRE(out && q && scale && ldo >= C && ldq >= C && ldq % 16 == 0 && hgv_aligned(q, 16), HGV_EINVAL,
                "unpack8: null / misaligned buffer or bad leading dimension");
    const int nb = (C + 31) / 32;
    HGV_REQUIRE(nb <= 32 * 65535, HGV_EUNSUPPORTED, "unpack8: too many columns");
    const P8Grid g = p8_grid(N, nb);
    const bool vec = hgv_aligned(out, 16) && ldo % 4 == 0 && ldo >= (C + 3) / 4 * 4;
    if (vec) hipLaunchKernelGGL(k_unpack8<true>, g.grid, dim3(256), 0, stream, q, ldq, scale, nb, N, C, out, ldo, g.per_pass, g.rows);
    else hipLaunchKernelGGL(k_unpack8<false>, g.grid, dim3(256), 0, stream, q, ldq, scale, nb, N, C, out, ldo, g.per_pass, g.rows);
    HGV_CHECK_LAUNCH("unpack8");
    return HGV_OK;
}

// ---- weight gradient from the 8-bit form -----------------------------------------------------------------------------------------
// GW[N, K] = G^T V, V the values of an 8-bit matrix, with the column sums of G as the bias gradient.  V is exact in bf16, so three
// bf16 pieces of G (8 bits each, cut: together all 24) make the product exact up to its fp32 accumulation: three piece products
// where two fp32 operands take six.
//
// The matrix cores' sums are cut downwards, whatever their sign: over 1.28 M rows whose terms cancel that alone is 1.3e-6 of the result, and
// 4e-6 of the column sums of a gradient with a mean.  So a tile's sum starts from zero, every other tile holds -G and is subtracted, which
// leaves as many cuts upwards, and tiles are added in fp32 by eight and then to a second sum: 1e-7, for 5 % of the kernel's time.
//
// A workgroup takes 144 x 144 outputs over every sets-th tile of 32 rows: G is split and V widened on the way into LDS (row-major,
// 288 bytes per row, which spreads the eight rows of a transposing load over all banks), two buffers.  Wave w of nine owns columns
// 16 w .. of G and all columns of V; the column sums are a product with a tile of ones.  Six more waves load and split, so that this
// runs beside the products.  Partial sums are added in fp64 in a fixed order by k_tn8_reduce.
// 1.28 M rows, 138 x 138: 237 us = 3.8 TB/s (one sum in the matrix cores 224;  before that, nine waves that split and multiply in turn 260, with four movers 227; the six-product
// kernel over the unpacked matrix 400, and 165 for unpacking).  Three or four tiles in flight instead of two: 241 and 235.
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int T8_ROWS = 32, T8_W = 144, T8_LINE = 2 * T8_W, T8_PIECE = T8_ROWS * T8_LINE, T8_BUF = 4 * T8_PIECE, T8_LDS = 2 * T8_BUF + T8_ROWS * 32;
constexpr int T8_MOVERS = 384, T8_THREADS = 576 + T8_MOVERS, T8_Q = T8_ROWS * (T8_W / 4) / T8_MOVERS;      // three quads of four columns per mover and tile
constexpr int T8_SET = (81 + 9) * 256;                          // floats of a partial set: 81 tiles, nine tiles of column sums

struct Tn8Args {
    const float* G; int64_t ldg; int N;
    const int8_t* q; int64_t ldq; const uint8_t* scale; int nb, K;
    int64_t M, steps;
    int ngrps, kgrps, sets;
    float* partial;                                             // [n group][k group][set][T8_SET]
};

__device__ __forceinline__ uint2 t8_pack(const uint32_t b[4]) {  // upper halves of four floats
    return make_uint2(__builtin_amdgcn_perm(b[1], b[0], 0x07060302u), __builtin_amdgcn_perm(b[3], b[2], 0x07060302u));
}

__device__ __forceinline__ bf16x8 t8_read(const unsigned char* p, int line = T8_LINE) {
    typedef __attribute__((address_space(3))) s16x4 lds_v;
    union { struct { s16x4 a, b; } s; bf16x8 v; } u;
    u.s.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v*)p);
    u.s.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v*)(p + 16 * line));
    return u.v;
}

// Waves 0 ... 8 multiply, waves 9 ... 14 move: between two barriers the products of a tile run beside the splitting of the next one
// and the loads of the one after that.
__global__ __launch_bounds__(T8_THREADS) void k_gemm_tn8(const Tn8Args a) {
    extern __shared__ __align__(16) unsigned char t8_lds[];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int per = a.ngrps * a.kgrps, grp = blockIdx.x % per, set = blockIdx.x / per;
    const int ng = grp / a.kgrps, kg = grp - ng * a.kgrps;
    const int n0 = T8_W * ng, k0 = T8_W * kg, n_w = min(T8_W, a.N - n0), k_w = min(T8_W, a.K - k0);
    const int nt = (n_w + 15) / 16, kt = (k_w + 15) / 16;
    // tiles set, set + sets, ...; the intervals are a multiple of two (the slot of a tile is a compile-time index), past the end the
    // movers bring the last tile again and nobody multiplies it
    const int64_t mine = (a.steps - set + a.sets - 1) / a.sets, intervals = (mine + 1) / 2 * 2, last = mine - 1;
    // a tile of ones behind the two buffers, for the column sums
    for (int i = t; i < T8_ROWS * 4; i += T8_THREADS) *(uint2*)(t8_lds + 2 * T8_BUF + i * 8) = make_uint2(0x3f803f80u, 0x3f803f80u);
    if (wave < 9) {
        f32x4 acc[9], accb = {0.f, 0.f, 0.f, 0.f}, sum[9], sumb = {0.f, 0.f, 0.f, 0.f};       // of up to eight tiles; of all before them
#pragma unroll
        for (int k = 0; k < 9; ++k) acc[k] = sum[k] = f32x4{0.f, 0.f, 0.f, 0.f};
        const int i16 = lane & 15;
        const int at = (4 * (lane >> 4) + (i16 >> 2)) * T8_LINE + (i16 & 3) * 8;
        __syncthreads();
        for (int64_t it = 0; it < intervals; ++it) {
            if (it < mine && wave < nt) {
                const unsigned char* base = t8_lds + (it & 1) * T8_BUF + at;
                const float sign = (it & 1) ? -1.f : 1.f;
                bf16x8 gf[3];
#pragma unroll
                for (int j = 0; j < 3; ++j) gf[j] = t8_read(base + j * T8_PIECE + wave * 32);
#pragma unroll
                for (int k = 0; k < 9; ++k)
                    if (k < kt) {
                        const bf16x8 v = t8_read(base + 3 * T8_PIECE + k * 32);
                        f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int j = 2; j >= 0; --j) t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(gf[j], v, t, 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[k][i] = fmaf(t[i], sign, acc[k][i]);
                    }
                if (kg == 0) {
                    const bf16x8 ones = t8_read(t8_lds + 2 * T8_BUF + (4 * (lane >> 4) + (i16 >> 2)) * 32 + (i16 & 3) * 8, 32);
                    f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int j = 2; j >= 0; --j) t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(gf[j], ones, t, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; ++i) accb[i] = fmaf(t[i], sign, accb[i]);
                }
            }
            if ((it & 7) == 7) {
#pragma unroll
                for (int k = 0; k < 9; ++k) { sum[k] += acc[k]; acc[k] = f32x4{0.f, 0.f, 0.f, 0.f}; }
                sumb += accb; accb = f32x4{0.f, 0.f, 0.f, 0.f};
            }
            __syncthreads();
        }
        if (wave < nt) {
            float* out = a.partial + ((int64_t)grp * a.sets + set) * T8_SET + lane * 4;
#pragma unroll
            for (int k = 0; k < 9; ++k)
                if (k < kt) *(f32x4*)(out + (wave * 9 + k) * 256) = sum[k] + acc[k];
            if (kg == 0) *(f32x4*)(out + (81 + wave) * 256) = sumb + accb;
        }
    } else {
        // quads m, m + 384, m + 768 of the tile's 32 x 36.  One offset per quad; what depends on the tile is uniform; quads outside the
        // matrices read their first columns or last row and count as zeros.
        const int m = t - 9 * 64;
        uint32_t go[T8_Q], qo[T8_Q], so[T8_Q];
        int row[T8_Q], to[T8_Q];
        bool g_live[T8_Q], v_live[T8_Q];
#pragma unroll
        for (int i = 0; i < T8_Q; ++i) {
            const int f = m + T8_MOVERS * i, c = 4 * (f % (T8_W / 4));
            row[i] = f / (T8_W / 4);
            g_live[i] = c < n_w; v_live[i] = c < k_w;
            go[i] = (uint32_t)(g_live[i] ? c : 0); qo[i] = (uint32_t)(v_live[i] ? c : 0);
            so[i] = (k0 + qo[i]) >> 5;
            to[i] = row[i] * T8_LINE + 2 * c;
        }
        f32x4 g[2][T8_Q];
        uint32_t w[2][T8_Q];
        int by[2][T8_Q];
        auto load = [&](auto slot, int64_t it) __attribute__((always_inline)) {
            constexpr int S = decltype(slot)::value;
            const int64_t r0 = (set + min(it, last) * a.sets) * T8_ROWS;
            const int rows = (int)min(a.M - r0, (int64_t)T8_ROWS);          // 1 ... 32
            const float* gp = a.G + r0 * a.ldg + n0;
            const int8_t* qp = a.q + r0 * a.ldq + k0;
            const uint8_t* sp = a.scale + r0 * a.nb;
#pragma unroll
            for (int i = 0; i < T8_Q; ++i) {
                const int r = min(row[i], rows - 1);
                g[S][i] = *(const f32x4*)(gp + (uint32_t)(r * (int)a.ldg) + go[i]);
                w[S][i] = *(const uint32_t*)(qp + (uint32_t)(r * (int)a.ldq) + qo[i]);
                by[S][i] = sp[(uint32_t)(r * a.nb) + so[i]];
            }
        };
        auto put = [&](auto slot, int64_t it) __attribute__((always_inline)) {
            constexpr int S = decltype(slot)::value;
            unsigned char* base = t8_lds + (it & 1) * T8_BUF;
            const int rows = (int)min(a.M - (set + min(it, last) * a.sets) * T8_ROWS, (int64_t)T8_ROWS);
#pragma unroll
            for (int i = 0; i < T8_Q; ++i) asm volatile("" : "+v"(g[S][i]), "+v"(w[S][i]), "+v"(by[S][i]));      // used from here on
#pragma unroll
            for (int i = 0; i < T8_Q; ++i) {
                const bool in = row[i] < rows, gi = in && g_live[i], vi = in && v_live[i];
                uint32_t p[3][4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float x = gi ? (S ? -g[S][i][e] : g[S][i][e]) : 0.f;
                    p[0][e] = __float_as_uint(x);
                    const float r = x - __uint_as_float(p[0][e] & 0xffff0000u);              // exact
                    p[1][e] = __float_as_uint(r);
                    p[2][e] = __float_as_uint(r - __uint_as_float(p[1][e] & 0xffff0000u));  // exact, eight bits left
                }
                float v[4];
                p8_values4(vi ? w[S][i] : 0u, vi ? by[S][i] : 127, v);
                const uint32_t vb[4] = {__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
                unsigned char* at = base + to[i];
#pragma unroll
                for (int j = 0; j < 3; ++j) *(uint2*)(at + j * T8_PIECE) = t8_pack(p[j]);
                *(uint2*)(at + 3 * T8_PIECE) = t8_pack(vb);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        constexpr std::integral_constant<int, 0> S0{};
        constexpr std::integral_constant<int, 1> S1{};
        load(S0, 0);
        load(S1, 1);
        put(S0, 0);
        __syncthreads();
        for (int64_t it = 0; it < intervals; it += 2) {
            load(S0, it + 2);
            __builtin_amdgcn_sched_barrier(0);
            put(S1, it + 1);
            __syncthreads();
            load(S1, it + 3);
            __builtin_amdgcn_sched_barrier(0);
            put(S0, it + 2);
            __syncthreads();
        }
    }
}

// One workgroup per 64 floats of a tile: 16 threads' worth of sets per float, added in a fixed order.
__global__ __launch_bounds__(1024) void k_tn8_reduce(const float* __restrict__ partial, const int sets, const int ngrps, const int kgrps, const int N,
                                                     const int K, float* __restrict__ GW, const int64_t ldgw, float* __restrict__ gbias) {
    __shared__ double red[1024];
    const int grp = blockIdx.y, ng = grp / kgrps, kg = grp - ng * kgrps;
    const int tile = blockIdx.x >> 2, part = blockIdx.x & 3;
    const bool bias = tile >= 81;
    const int tn = bias ? tile - 81 : tile / 9, tk = bias ? 0 : tile - 9 * tn;
    const int n0 = T8_W * ng + 16 * tn, k0 = T8_W * kg + 16 * tk;
    if (n0 >= N || (bias ? kg != 0 || !gbias : k0 >= K) || 16 * tn >= T8_W) return;      // the whole workgroup
    const int e = threadIdx.x & 63, j = threadIdx.x >> 6;
    const float* p = partial + (int64_t)grp * sets * T8_SET + tile * 256 + part * 64 + e;
    double s = 0.0;
#pragma unroll 8
    for (int i = j; i < sets; i += 16) s += (double)p[(int64_t)i * T8_SET];
    red[threadIdx.x] = s;
    for (int o = 8; o > 0; o >>= 1) {
        __syncthreads();
        if (j < o) red[threadIdx.x] += red[threadIdx.x + 64 * o];
    }
    if (j > 0) return;
    const int f = part * 64 + e, lane = f >> 2;                 // lane and register of the product's result
    const int n = n0 + 4 * (lane >> 4) + (f & 3), k = k0 + (lane & 15);
    if (n >= N) return;
    if (bias) {
        if ((lane & 15) == 0) gbias[n] = (float)red[e];
    } else if (k < K) {
        GW[(int64_t)n * ldgw + k] = (float)red[e];
    }
}

int tn8_sets(int64_t M, int per) {
    const int64_t steps = hgv_cdiv(M, T8_ROWS);
    // one workgroup per compute unit, at least four tiles each
    return (int)max((int64_t)1, min((int64_t)max(256 / per, 1), steps / 4));
}

}  // namespace

extern "C" size_t hgv_gemm_tn8_ws(int64_t M, int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    const int per = (int)(hgv_cdiv(N, T8_W) * hgv_cdiv(K, T8_W));
    return hgv_align256((size_t)per * tn8_sets(M, per) * T8_SET * sizeof(float));
}

extern "C" int hgv_gemm_tn8(const float* G, int64_t ldg, int N, const int8_t* q, int64_t ldq, const uint8_t* scale, int K, int64_t M, float* GW,
                            int64_t ldgw, float* gbias, void* ws, size_t ws_bytes, hipStream_t stream) {
    HGV_REQUIRE(M > 0 && N > 0 && K > 0, HGV_EINVAL, "gemm_tn8: bad sizes");
    HGV_REQUIRE(G && q && scale && GW && hgv_aligned(G, 16) && ldg % 4 == 0 && ldg >= (N + 3) / 4 * 4 && ldq >= K && ldq % 16 == 0 &&
                hgv_aligned(q, 16) && ldgw >= K, HGV_EINVAL, "gemm_tn8: null / misaligned buffer or bad leading dimension");
    HGV_REQUIRE(N <= 65536 && K <= 65536, HGV_EUNSUPPORTED, "gemm_tn8: widths above 65536");
    HGV_REQUIRE(ws && ws_bytes >= hgv_gemm_tn8_ws(M, N, K) && hgv_aligned(ws, 256), HGV_EWORKSPACE, "gemm_tn8: workspace too small or misaligned");
    Tn8Args a = {};
    a.G = G; a.ldg = ldg; a.N = N; a.q = q; a.ldq = ldq; a.scale = scale; a.nb = (K + 31) / 32; a.K = K; a.M = M;
    a.steps = hgv_cdiv(M, T8_ROWS); a.ngrps = (int)hgv_cdiv(N, T8_W); a.kgrps = (int)hgv_cdiv(K, T8_W);
    const int per = a.ngrps * a.kgrps;
    a.sets = tn8_sets(M, per); a.partial = (float*)ws;
    HGV_REQUIRE(per <= 65535, HGV_EUNSUPPORTED, "gemm_tn8: widths not supported");
    static bool raised[64] = {false};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) dev = 0;
    if (!raised[dev]) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k_gemm_tn8), hipFuncAttributeMaxDynamicSharedMemorySize, T8_LDS);
        HGV_REQUIRE(e == hipSuccess, HGV_ELAUNCH, "gemm_tn8: cannot raise the dynamic LDS limit: %s", hipGetErrorString(e));
        raised[dev] = true;
    }
    hipLaunchKernelGGL(k_gemm_tn8, dim3((unsigned)(per * a.sets)), dim3(T8_THREADS), T8_LDS, stream, a);
    hipLaunchKernelGGL(k_tn8_reduce, dim3(90 * 4, (unsigned)per), dim3(1024), 0, stream, a.partial, a.sets, a.ngrps, a.kgrps, N, K, GW, ldgw, gbias);
    HGV_CHECK_LAUNCH("gemm_tn8");
    return HGV_OK;
}
