/* The FP8-128 encoding of a block's values, for the kernels that write it. */
#pragma once

#include "k3_device.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace k3 {

constexpr uint32_t kBlock = 128;      /* values of a block */
constexpr float kTop = 448.0f;        /* largest e4m3 */
constexpr float kLeast = 0x1.cp-118f; /* 448 * 2^-126 */

/* Scale and its inverse of a block with maximum a. */
__device__ __forceinline__ void fp8_scales(float a, float &scale, float &inv) {
    a = fmaxf(a, kLeast);
    scale = __fdiv_rn(a, kTop);
    inv = __fdiv_rn(kTop, a);
}

/* Eight values as codes. v inv is at most 448 (1 + 2^-23), which rounds to
 * 448; NaN (and inf x 0) gives a NaN code. */
__device__ __forceinline__ uint2 fp8_codes8(const float (&v)[8], float inv) {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const float *u = v + 4 * h;
        w[h] = e4m3x2_raw<true>(__fmul_rn(u[2], inv), __fmul_rn(u[3], inv),
                                e4m3x2_raw<false>(__fmul_rn(u[0], inv), __fmul_rn(u[1], inv), 0u));
    }
    return make_uint2(w[0], w[1]);
}

__device__ __forceinline__ void unpack8(const uint4 &p, float (&v)[8]) {
    const uint32_t d[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[2 * i] = bf16_lo(d[i]);
        v[2 * i + 1] = bf16_hi(d[i]);
    }
}
__device__ __forceinline__ void load8(const uint16_t *src, float (&v)[8]) {
    unpack8(*(const uint4 *)src, v);
}

__device__ __forceinline__ float max8(const float (&v)[8]) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(v[i]));
    return m;
}

}  // namespace k3
