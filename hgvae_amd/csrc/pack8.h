// The 8-bit form of activation checkpoints (see pack8.hip), for the kernels that write or read it.
#pragma once
#include "common.h"

extern "C" int hgv_pack8(const float* x, int64_t ldx, int64_t N, int C, int8_t* q, int64_t ldq, uint8_t* scale, hipStream_t stream);

// Byte of a block from the bits of its largest magnitude (compared as integers: a NaN or infinity wins).
__device__ __forceinline__ int p8_byte(uint32_t amax) {
    const int field = (int)(amax >> 23);
    if (field == 255) return 255;
    // 127.5 * 2^e = 1.9921875 * 2^(e + 6): the mantissa field alone decides.  e stays at 121: 128 * 2^121 would not be finite
    return min(max(field - 6 + ((amax & 0x7fffffu) >= 0x7f0000u ? 1 : 0), 1), 248);
}

__device__ __forceinline__ uint32_t p8_max8(uint32_t v) {       // over the eight lanes of a block
    v = max(v, (uint32_t)__shfl_xor((int)v, 1, 64));
    v = max(v, (uint32_t)__shfl_xor((int)v, 2, 64));
    return max(v, (uint32_t)__shfl_xor((int)v, 4, 64));
}

// Four integers of a block as bytes.  x * 2^-e + 1.5 * 2^23 in one rounding: the low byte of the sum's bits is round_to_nearest_even
// (x * 2^-e) in two's complement (|q| < 2^22), so a value takes two instructions: the cut to 127 * 2^e, which only bites beyond
// 127.5 * 2^121, and the multiply-add.
__device__ __forceinline__ uint32_t p8_quantise4(const float v[4], int byte) {
    const float inv = __uint_as_float((uint32_t)(254 - byte) << 23);            // 2^-e, e = byte - 127 in [-126, 121]
    const float lim = __uint_as_float(((uint32_t)(byte + 6) << 23) | 0x7e0000u);  // 127 * 2^e
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(fmaf(__builtin_amdgcn_fmed3f(v[i], -lim, lim), inv, 12582912.f));
    const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0c);
    return byte == 255 ? 0u : lo | hi;
}

__device__ __forceinline__ float p8_step(int byte) {                               // 2^e, or NaN
    return __uint_as_float(byte == 255 ? 0x7fc00000u : (uint32_t)byte << 23);
}

__device__ __forceinline__ void p8_values4(uint32_t w, int byte, float v[4]) {
    const float step = p8_step(byte);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (float)(int)(int8_t)(w >> (8 * i)) * step;
}
