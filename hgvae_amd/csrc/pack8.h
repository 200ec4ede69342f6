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

__device__ __forceinline__ uint32_t p8_quantise4(const float v[4], int byte) {
    if (byte == 255) return 0;
    const float inv = __uint_as_float((uint32_t)(254 - byte) << 23);            // 2^-e, e = byte - 127 in [-126, 121]
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= ((uint32_t)(int)fminf(fmaxf(rintf(v[i] * inv), -127.f), 127.f) & 255u) << (8 * i);
    return w;
}

__device__ __forceinline__ float p8_step(int byte) {                               // 2^e, or NaN
    return __uint_as_float(byte == 255 ? 0x7fc00000u : (uint32_t)byte << 23);
}

__device__ __forceinline__ void p8_values4(uint32_t w, int byte, float v[4]) {
    const float step = p8_step(byte);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (float)(int)(int8_t)(w >> (8 * i)) * step;
}
