/*
 * The gated activation of the routed experts' gate/up rows times their route
 * weights, and its gradient. No reference counterpart (the reference only
 * serves); the formulas are in include/k3_moe.h.
 *
 * A wave a row: each lane takes eight columns at a time of gate and of up, so
 * every load and store is 16 bytes, and the gradient by the route's weight is one sum over
 * the wave. Bound by memory: 6 bytes a value forward, 10 backward. 32768 rows of F = 2048: 67 and 114
 * us, 6.0 and 5.9 TB/s, where a large copy moves 5.2; 222 rows of F = 1024 4 and 6 us, a wave's
 * latency.
 */
#include "k3_device.h"
#include "k3_fp8.h"
#include "k3_internal.h"
#include "../../include/k3_moe.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace k3 {
namespace {

constexpr uint32_t kMostFfn = 1u << 15, kMostRows = 65535u * 32u;

struct GatedArgs {
    uint16_t *out;               /* h, or the gradient of gate/up */
    float *weight_gradient;      /* [routes], or NULL */
    const uint16_t *dh, *gate_up;
    const uint32_t *offsets, *route_index;
    const float *route_weights;
    uint32_t R, routes, E, F;
    float beta, linear, by, by_linear; /* SiTU's bounds and their reciprocals */
};

/* sigmoid(g) and 1 - sigmoid(g), each to a few ulps of itself (0 where it is under 2^-126): of e^-|g|,
 * so that neither is the difference of numbers near 1. */
__device__ __forceinline__ void sigmoids(float g, float &s, float &rest) {
    const float e = __builtin_amdgcn_exp2f(__fmul_rn(fabsf(g), -1.44269504088896341f));
    const float big = __builtin_amdgcn_rcpf(__fadd_rn(1.0f, e)), small = __fmul_rn(e, big);
    s = g < 0.0f ? small : big;
    rest = g < 0.0f ? big : small;
}
/* 1 - tanh(y)^2, t = tanh(y): 4 e / (1 + e)^2 with e = e^-2|y| where that would cancel. */
__device__ __forceinline__ float tanh_slope(float y, float t) {
    const float e = __builtin_amdgcn_exp2f(__fmul_rn(fabsf(y), -2.88539008177792681f));
    const float r = __builtin_amdgcn_rcpf(__fadd_rn(1.0f, e));
    return fabsf(y) < 0.25f ? fmaf(-t, t, 1.0f) : __fmul_rn(__fmul_rn(4.0f, e), __fmul_rn(r, r));
}

/* act(g, u), and with Slopes its derivatives by g and u. In fp32 on the hardware's
 * exp2 and reciprocal (1 ulp): what comes of them is rounded to bf16, or summed. */
template <bool SWIGLU, bool Slopes>
__device__ __forceinline__ float gated_value(float g, float u, const GatedArgs &A, float &by_g,
                                             float &by_u) {
    float s, rest;
    sigmoids(g, s, rest);
    if constexpr (SWIGLU) {
        const float gs = __fmul_rn(g, s);
        if (Slopes) {
            by_g = __fmul_rn(__fmul_rn(s, fmaf(g, rest, 1.0f)), u);
            by_u = gs;
        }
        return __fmul_rn(gs, u);
    } else {
        const float yg = __fmul_rn(g, A.by), yu = __fmul_rn(u, A.by_linear);
        const float tg = tanh_f32(yg), tu = tanh_f32(yu);
        const float a = __fmul_rn(A.beta, tg), c = __fmul_rn(A.linear, tu), as = __fmul_rn(a, s);
        if (Slopes) {
            by_g = __fmul_rn(__fmul_rn(s, fmaf(a, rest, tanh_slope(yg, tg))), c);
            by_u = __fmul_rn(as, tanh_slope(yu, tu));
        }
        return __fmul_rn(as, c);
    }
}

/* Past the caches: 16384 rows of 2 x 1024 19.5 and 16.5 us, 32768 rows of 2 x 3584 133 and 130. */
__device__ __forceinline__ void store8(uint16_t *to, const float (&v)[8]) {
    const u32x4_t packed{bf16_pack2(v[0], v[1]), bf16_pack2(v[2], v[3]), bf16_pack2(v[4], v[5]),
                         bf16_pack2(v[6], v[7])};
    __builtin_nontemporal_store(packed, (u32x4_t *)to);
}

/* The wave's row, its route (routes: none) and weight; false past the last expert's rows. */
__device__ __forceinline__ bool wave_row(const GatedArgs &A, uint32_t &row, uint32_t &route, float &w) {
    row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4u + (threadIdx.x >> 6));
    if (row >= min(A.R, A.offsets[A.E])) return false;
    route = A.route_index ? A.route_index[row] : row;
    if (route > A.routes) route = A.routes;
    w = !A.route_weights ? 1.0f : route < A.routes ? A.route_weights[route] : 0.0f;
    return true;
}

template <bool SWIGLU>
__global__ __launch_bounds__(256) void gated_kernel(GatedArgs A) {
    uint32_t row, route;
    float w;
    if (!wave_row(A, row, route, w)) return;
    const uint16_t *gate = A.gate_up + 2u * (uint64_t)row * A.F, *up = gate + A.F;
    uint16_t *out = A.out + (uint64_t)row * A.F;
    for (uint32_t c = 8u * (threadIdx.x & 63u); c < A.F; c += 512u) {
        float g[8], u[8], unused;
        load8(gate + c, g);
        load8(up + c, u);
#pragma unroll
        for (int i = 0; i < 8; i++)
            g[i] = __fmul_rn(w, gated_value<SWIGLU, false>(g[i], u[i], A, unused, unused));
        store8(out + c, g);
    }
}

template <bool SWIGLU>
__global__ __launch_bounds__(256) void gated_backward_kernel(GatedArgs A) {
    uint32_t row, route;
    float w, sum = 0.0f;
    if (!wave_row(A, row, route, w)) return;
    const uint64_t at = 2u * (uint64_t)row * A.F;
    const uint16_t *gate = A.gate_up + at, *up = gate + A.F, *dh = A.dh + (uint64_t)row * A.F;
    uint16_t *dgate = A.out + at, *dup = dgate + A.F;
    for (uint32_t c = 8u * (threadIdx.x & 63u); c < A.F; c += 512u) {
        float g[8], u[8], d[8];
        load8(gate + c, g);
        load8(up + c, u);
        load8(dh + c, d);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float by_g, by_u;
            const float value = gated_value<SWIGLU, true>(g[i], u[i], A, by_g, by_u);
            sum = fmaf(d[i], value, sum);
            const float dw = __fmul_rn(d[i], w);
            g[i] = __fmul_rn(dw, by_g);
            u[i] = __fmul_rn(dw, by_u);
        }
        store8(dgate + c, g);
        store8(dup + c, u);
    }
    if (!A.weight_gradient) return;
    sum = wave_sum(sum);
    if ((threadIdx.x & 63u) == 0u && route < A.routes) A.weight_gradient[route] = sum;
}

/* Routes without a row (repeated ones, ids of no expert) have gradient 0. A kernel, as
 * a captured memset has given wrong results on replays. */
__global__ __launch_bounds__(256) void zero_kernel(float *__restrict__ to, uint32_t n) {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i < n) to[i] = 0.0f;
}

/* Whether an output lies over what rows are found by, or over the route weights. */
bool over_routes(const void *output, uint64_t bytes, const GatedArgs &A) {
    return overlap(output, bytes, A.offsets, 4u * (uint64_t)(A.E + 1u)) ||
           (A.route_index && overlap(output, bytes, A.route_index, 4u * (uint64_t)A.R)) ||
           (A.route_weights && overlap(output, bytes, A.route_weights, 4u * (uint64_t)A.routes));
}

bool gated_args(GatedArgs &A, const void *gate_up, const uint32_t *offsets, const uint32_t *route_index,
                const float *route_weights, uint32_t rows, uint32_t routes, uint32_t experts, uint32_t ffn,
                uint32_t activation, float beta, float linear_beta) {
    if (!gate_up || (uintptr_t)gate_up % 16u != 0u || !offsets ||
        (((uintptr_t)offsets | (uintptr_t)route_index | (uintptr_t)route_weights) % 4u) != 0u || rows == 0u ||
        rows > kMostRows || routes > kMostRows || (route_weights && routes == 0u) || experts == 0u ||
        experts > 1024u || ffn == 0u || ffn % 8u != 0u || ffn > kMostFfn || activation > 1u ||
        (activation == K3_MOE_ACT_SITU && !(beta > 0.0f && linear_beta > 0.0f)))
        return false;
    const auto inverse = [](float v) { return v < 0x1p-127f ? 0x1.fffffep127f : 1.0f / v; };
    A.gate_up = (const uint16_t *)gate_up, A.offsets = offsets, A.route_index = route_index;
    A.route_weights = route_weights, A.R = rows, A.routes = routes, A.E = experts, A.F = ffn;
    A.beta = beta, A.linear = linear_beta, A.by = inverse(beta), A.by_linear = inverse(linear_beta);
    return true;
}

}  // namespace
}  // namespace k3

using namespace k3;

extern "C" bool k3_moe_gated_rows_bf16(void *output, const void *gate_up, const uint32_t *offsets,
                                       const uint32_t *route_index, const float *route_weights,
                                       uint32_t rows, uint32_t routes, uint32_t expert_count,
                                       uint32_t ffn, uint32_t activation, float beta,
                                       float linear_beta, void *stream) {
    GatedArgs A{};
    const uint64_t bytes = 2u * (uint64_t)rows * ffn;
    if (!output || (uintptr_t)output % 16u != 0u ||
        !gated_args(A, gate_up, offsets, route_index, route_weights, rows, routes, expert_count, ffn, activation,
                    beta, linear_beta) ||
        overlap(output, bytes, gate_up, 2u * bytes) || over_routes(output, bytes, A))
        return false;
    A.out = (uint16_t *)output;
    const auto kernel = activation == K3_MOE_ACT_SWIGLU ? gated_kernel<true> : gated_kernel<false>;
    hipLaunchKernelGGL(kernel, dim3((rows + 3u) / 4u), dim3(256), 0, (hipStream_t)stream, A);
    return hipGetLastError() == hipSuccess;
}

extern "C" bool k3_moe_gated_rows_backward_bf16(void *gate_up_gradient, float *weight_gradient,
                                                const void *output_gradient, const void *gate_up,
                                                const uint32_t *offsets, const uint32_t *route_index,
                                                const float *route_weights, uint32_t rows,
                                                uint32_t routes, uint32_t expert_count, uint32_t ffn,
                                                uint32_t activation, float beta, float linear_beta,
                                                void *stream) {
    GatedArgs A{};
    const uint64_t bytes = 2u * (uint64_t)rows * ffn, grads = 4u * (uint64_t)routes;
    if (!gate_up_gradient || !output_gradient ||
        (((uintptr_t)gate_up_gradient | (uintptr_t)output_gradient) % 16u) != 0u ||
        (uintptr_t)weight_gradient % 4u != 0u || (weight_gradient && routes == 0u) ||
        !gated_args(A, gate_up, offsets, route_index, route_weights, rows, routes, expert_count, ffn, activation,
                    beta, linear_beta) ||
        /* each value's place is read by the lane that writes there: the gradient may take gate_up's */
        (gate_up_gradient != gate_up && overlap(gate_up_gradient, 2u * bytes, gate_up, 2u * bytes)) ||
        overlap(gate_up_gradient, 2u * bytes, output_gradient, bytes) ||
        over_routes(gate_up_gradient, 2u * bytes, A) ||
        (weight_gradient && (overlap(weight_gradient, grads, gate_up_gradient, 2u * bytes) ||
                             overlap(weight_gradient, grads, gate_up, 2u * bytes) ||
                             overlap(weight_gradient, grads, output_gradient, bytes) ||
                             over_routes(weight_gradient, grads, A))))
        return false;
    A.out = (uint16_t *)gate_up_gradient, A.weight_gradient = weight_gradient;
    A.dh = (const uint16_t *)output_gradient;
    const hipStream_t st = (hipStream_t)stream;
    if (weight_gradient) {
        hipLaunchKernelGGL(zero_kernel, dim3((routes + 255u) / 256u), dim3(256), 0, st, weight_gradient, routes);
        if (hipGetLastError() != hipSuccess) return false;
    }
    const auto kernel =
        activation == K3_MOE_ACT_SWIGLU ? gated_backward_kernel<true> : gated_backward_kernel<false>;
    hipLaunchKernelGGL(kernel, dim3((rows + 3u) / 4u), dim3(256), 0, st, A);
    return hipGetLastError() == hipSuccess;
}
