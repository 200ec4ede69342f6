// Activation checkpoints in 8 bits: a row-major fp32 matrix as 8-bit integers with one power of two for each row and block
// of 32 columns, and back.
//
// For a block with largest magnitude amax:  e = floor(log2 amax) - 6, one more where amax >= 127.5 * 2^e, held in [-126, 121];
// q = round_to_nearest_even(x * 2^-e), |q| <= 127 (cut only beyond 127.5 * 2^121); the stored byte is e + 127 and the value that stands for x is q * 2^e.
// A power of two makes both products exact (so the quotient is the same in any precision), and q * 2^e has at most 7
// significant bits: it is exact in bf16 too, which is what the weight gradient reads.  |value - x| <= 2^(e-1) <= amax / 126
// for amax >= 2^-120.  A block that holds an infinity or a NaN gets the byte 255 and reads back as NaN.
#include "pack8.h"

namespace {

__device__ __forceinline__ uint32_t max8(uint32_t v) {          // over the eight lanes of a block
    v = max(v, (uint32_t)__shfl_xor((int)v, 1, 64));
    v = max(v, (uint32_t)__shfl_xor((int)v, 2, 64));
    return max(v, (uint32_t)__shfl_xor((int)v, 4, 64));
}

// Eight lanes take one block of 32 columns of one row (a lane four columns); the 32 lane groups of a workgroup cover
// floor(32 / blocks) rows at a time (wide matrices: 32 blocks of one row, further blocks in blockIdx.y), and walk rows with
// that stride.  Bound by memory: 4 bytes read and 1.03 written per element.
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
        const int byte = p8_byte(max8(m));
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
        if (VEC) *(float4*)p = make_float4(v[0], v[1], v[2], v[3]);       // bytes behind the last column are zero
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
