/*
 * FP8-128: e4m3 codes with an fp32 scale for each block of 128 (128 values of
 * a token row, 128 x 128 of a weight), the product of such rows and weights,
 * and the routed experts on it. No reference counterpart; the encoding and the
 * products are defined in include/k3_moe.h.
 *
 *   rows_kernel       token rows (bf16, or fp32 for the experts' activation)
 *   weight_kernel     a weight, one 128 x 128 block a block
 *   product_kernel    output = rows . weight, 16 tokens x 16 rows a wave
 *   gateup_kernel     act(gate . x, up . x) of every selected expert's rows
 *   down_kernel       y[route] = bf16(down . h)
 *
 * MFMA operands (V_MFMA_F32_16X16X128_F8F6F4): lane 16 g + c holds 32 codes of
 * row c of the 16 x 128 slices. Both operands take the bytes [32 g, 32 g + 32)
 * of their row there: whichever columns the unit takes them for, they are the
 * same in both, and the sum is over all. Weights are the first operand, tokens
 * the second: lane (g, c) of the result holds weight rows 4 g + i (i < 4) of
 * token c, so one factor scales all four.
 */
#include "k3_device.h"
#include "k3_fp8.h"
#include "k3_internal.h"
#include "../../include/k3_moe.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace k3 {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kBlock = 128;                /* values of a block */
constexpr float kTop = 448.0f;                  /* largest e4m3 */
constexpr float kLeast = 0x1.cp-118f;           /* 448 * 2^-126 */

inline size_t align256(size_t v) { return (v + 255u) & ~(size_t)255u; }

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

__device__ __forceinline__ void load8(const uint16_t *src, float (&v)[8]) {
    const uint4 p = *(const uint4 *)src;
    const uint32_t d[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[2 * i] = bf16_lo(d[i]);
        v[2 * i + 1] = bf16_hi(d[i]);
    }
}
__device__ __forceinline__ void load8(const float *src, float (&v)[8]) {
    const float4 a = ((const float4 *)src)[0], b = ((const float4 *)src)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

__device__ __forceinline__ float max8(const float (&v)[8]) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(v[i]));
    return m;
}

/* Sixteen lanes a block of 128 values, eight values a lane: one 16-byte load
 * (bf16), a maximum within a row of lanes, one 8-byte store. */
template <class S>
__global__ __launch_bounds__(256) void rows_kernel(uint8_t *__restrict__ codes,
                                                   float *__restrict__ scales,
                                                   const S *__restrict__ src, uint64_t blocks) {
    const uint64_t q = (uint64_t)blockIdx.x * 16u + (threadIdx.x >> 4);
    if (q >= blocks) return; /* whole rows of 16 lanes */
    const uint32_t l = threadIdx.x & 15u;
    float v[8], scale, inv;
    load8(src + kBlock * q + 8u * l, v);
    fp8_scales(row_group_max<16>(max8(v)), scale, inv);
    *(uint2 *)(codes + kBlock * q + 8u * l) = fp8_codes8(v, inv);
    if (l == 0u) scales[q] = scale;
}

/* One block of 256 threads a 128 x 128 block: thread t holds eight columns of
 * rows t / 16 + 16 m; rows past the last are left out. */
__global__ __launch_bounds__(256) void weight_kernel(uint8_t *__restrict__ codes,
                                                     float *__restrict__ scales,
                                                     const uint16_t *__restrict__ src,
                                                     uint32_t rows, uint32_t cols) {
    __shared__ float red[4];
    const uint32_t nb = cols / kBlock, b = blockIdx.x % nb, rb = blockIdx.x / nb;
    const uint32_t c = kBlock * b + 8u * (threadIdx.x & 15u), r0 = kBlock * rb + (threadIdx.x >> 4);
    float v[8][8], m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t r = r0 + 16u * (uint32_t)i;
#pragma unroll
        for (int j = 0; j < 8; j++) v[i][j] = 0.0f;
        if (r < rows) load8(src + (uint64_t)r * cols + c, v[i]);
        m = fmaxf(m, max8(v[i]));
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    if ((threadIdx.x & 63u) == 0u) red[threadIdx.x >> 6] = m;
    __syncthreads();
    float scale, inv;
    fp8_scales(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), scale, inv);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t r = r0 + 16u * (uint32_t)i;
        if (r < rows) *(uint2 *)(codes + (uint64_t)r * cols + c) = fp8_codes8(v[i], inv);
    }
    if (threadIdx.x == 0u) scales[blockIdx.x] = scale;
}

__device__ __forceinline__ f32x4 mfma_block(const uint4 &a0, const uint4 &a1, const uint4 &b0,
                                            const uint4 &b1) {
    const i32x8 a = {(int)a0.x, (int)a0.y, (int)a0.z, (int)a0.w,
                     (int)a1.x, (int)a1.y, (int)a1.z, (int)a1.w};
    const i32x8 b = {(int)b0.x, (int)b0.y, (int)b0.z, (int)b0.w,
                     (int)b1.x, (int)b1.y, (int)b1.z, (int)b1.w};
    /* both scale operands 2^0 */
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 0,
                                                            0, 0, 127, 0, 127);
}

/* acc += sum over the blocks of scale x (weight rows . token rows); w, x: this
 * lane's weight and token row, at byte 32 g of the first block. */
__device__ __forceinline__ void tile16(f32x4 &acc, const uint8_t *w, const float *sw,
                                       const uint8_t *x, const float *sx, uint32_t nblk) {
    for (uint32_t b = 0; b < nblk; b++, w += kBlock, x += kBlock) {
        const f32x4 p = mfma_block(((const uint4 *)w)[0], ((const uint4 *)w)[1],
                                   ((const uint4 *)x)[0], ((const uint4 *)x)[1]);
        const float s = __fmul_rn(sx[b], sw[b]);
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] = fmaf(p[i], s, acc[i]);
    }
}

__global__ __launch_bounds__(256) void product_kernel(uint16_t *__restrict__ out,
                                                      const uint8_t *__restrict__ codes,
                                                      const float *__restrict__ scales,
                                                      const uint8_t *__restrict__ xq,
                                                      const float *__restrict__ xs, uint32_t T,
                                                      uint32_t N, uint32_t K) {
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, c = lane & 15u, nblk = K / kBlock;
    const uint32_t n0 = 64u * blockIdx.x + 16u * (threadIdx.x >> 6), t0 = 16u * blockIdx.y;
    if (n0 >= N) return;
    const uint32_t n = min(n0 + c, N - 1u), t = min(t0 + c, T - 1u);
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    tile16(acc, codes + (uint64_t)n * K + 32u * g, scales + (uint64_t)(n0 / kBlock) * nblk,
           xq + (uint64_t)t * K + 32u * g, xs + (uint64_t)t * nblk, nblk);
#pragma unroll
    for (uint32_t i = 0; i < 4u; i++)
        if (t0 + c < T && n0 + 4u * g + i < N)
            out[(uint64_t)(t0 + c) * N + n0 + 4u * g + i] = f32_to_bf16(acc[i]);
}

/* ---------------------------------------------------------------------- */
/* experts                                                                 */
/* ---------------------------------------------------------------------- */

/* ids with a token's repeated ones invalidated, as the plan drops them. */
__global__ __launch_bounds__(256) void routes_kernel(uint32_t *__restrict__ out,
                                                     const uint32_t *__restrict__ ids, uint32_t T,
                                                     uint32_t k, uint32_t E) {
    const uint32_t t = blockIdx.x * 256u + threadIdx.x;
    if (t >= T) return;
    uint32_t e[32];
    token_routes<32>(ids, t, k, E, e);
#pragma unroll
    for (uint32_t r = 0; r < 32u; r++)
        if (r < k) out[(uint64_t)t * k + r] = e[r];
}

/* One block: the tiles {expert, first row, rows <= 16} in expert order. */
__global__ __launch_bounds__(1024) void tiles_kernel(uint32_t *__restrict__ tiles,
                                                     uint32_t *__restrict__ tile_count,
                                                     const uint32_t *__restrict__ counts,
                                                     const uint32_t *__restrict__ offsets,
                                                     uint32_t E) {
    __shared__ uint32_t tot[16];
    const uint32_t e = threadIdx.x, lane = e & 63u, wave = e >> 6;
    const uint32_t n = e < E ? counts[e] : 0u, mine = (n + 15u) / 16u;
    uint32_t inc = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t a = __shfl_up(inc, o, 64);
        if ((int)lane >= o) inc += a;
    }
    if (lane == 63u) tot[wave] = inc;
    __syncthreads();
    uint32_t at = inc - mine, total = 0u;
    for (uint32_t w = 0; w < 16u; w++) {
        if (w < wave) at += tot[w];
        total += tot[w];
    }
    for (uint32_t q = 0; q < mine; q++) {
        tiles[3u * (at + q)] = e;
        tiles[3u * (at + q) + 1u] = offsets[e] + 16u * q;
        tiles[3u * (at + q) + 2u] = min(16u, n - 16u * q);
    }
    if (e == 0u) *tile_count = total;
}

/* tanh to a few ulp: its odd series below 1/2, the exponential above. */
__device__ __forceinline__ float tanh_f32(float y) {
    const float a = fabsf(y), z = __fmul_rn(a, a);
    float p = -1.4558343870513183e-3f;
    p = fmaf(p, z, 3.5921280365724811e-3f);
    p = fmaf(p, z, -8.8632355299021966e-3f);
    p = fmaf(p, z, 2.1869488536155203e-2f);
    p = fmaf(p, z, -5.3968253968253968e-2f);
    p = fmaf(p, z, 1.3333333333333333e-1f);
    p = fmaf(p, z, -3.3333333333333333e-1f);
    const float lo = fmaf(__fmul_rn(a, z), p, a);
    const float e = __builtin_amdgcn_exp2f(__fmul_rn(a, 2.88539008177792681f)); /* e^2a */
    const float hi = fmaf(-2.0f, __builtin_amdgcn_rcpf(__fadd_rn(e, 1.0f)), 1.0f);
    return copysignf(a < 0.5f ? lo : hi, y);
}

/* The activation in fp32: it is encoded in e4m3 next, and exp2 and the
 * reciprocal of the hardware (1 ulp) are far inside that. */
__device__ __forceinline__ float act_f32(float g, float u, uint32_t kind, float beta, float lb) {
    const float e = __builtin_amdgcn_exp2f(__fmul_rn(g, -1.44269504088896341f));
    const float s = __builtin_amdgcn_rcpf(__fadd_rn(1.0f, e));
    if (kind == K3_MOE_ACT_SWIGLU) return __fmul_rn(__fmul_rn(g, s), u);
    const float bg = __fmul_rn(beta, tanh_f32(__fdiv_rn(g, beta)));
    const float bu = __fmul_rn(lb, tanh_f32(__fdiv_rn(u, lb)));
    return __fmul_rn(__fmul_rn(bg, s), bu);
}

struct ExpertArgs {
    const k3_moe_fp8_expert *experts;
    const uint32_t *tiles, *tile_count, *token_index, *route_index;
    const uint8_t *xq; /* [T, H] */
    const float *xs;
    float *h; /* [rows, F] in plan order */
    const uint8_t *hq;
    const float *hs;
    uint16_t *y; /* [routes, H] */
    uint32_t H, F, kind;
    float beta, lb;
};

__global__ __launch_bounds__(256) void gateup_kernel(ExpertArgs A) {
    if (blockIdx.y >= *A.tile_count) return;
    const uint32_t *tile = A.tiles + 3u * blockIdx.y;
    const uint32_t row0 = tile[1], rows = tile[2];
    const k3_moe_fp8_expert ex = A.experts[tile[0]];
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, c = lane & 15u, nblk = A.H / kBlock;
    const uint32_t f0 = 64u * blockIdx.x + 16u * (threadIdx.x >> 6);
    const uint32_t t = A.token_index[row0 + min(c, rows - 1u)];
    const uint64_t w = (uint64_t)(f0 + c) * A.H + 32u * g, sw = (uint64_t)(f0 / kBlock) * nblk;
    const uint8_t *x = A.xq + (uint64_t)t * A.H + 32u * g;
    const float *xs = A.xs + (uint64_t)t * nblk;
    f32x4 gate = {0.0f, 0.0f, 0.0f, 0.0f}, up = gate;
    tile16(gate, ex.gate_codes + w, ex.gate_scales + sw, x, xs, nblk);
    tile16(up, ex.up_codes + w, ex.up_scales + sw, x, xs, nblk);
    if (c >= rows) return;
#pragma unroll
    for (uint32_t i = 0; i < 4u; i++)
        A.h[(uint64_t)(row0 + c) * A.F + f0 + 4u * g + i] =
            act_f32(gate[i], up[i], A.kind, A.beta, A.lb);
}

__global__ __launch_bounds__(256) void down_kernel(ExpertArgs A) {
    if (blockIdx.y >= *A.tile_count) return;
    const uint32_t *tile = A.tiles + 3u * blockIdx.y;
    const uint32_t row0 = tile[1], rows = tile[2];
    const k3_moe_fp8_expert ex = A.experts[tile[0]];
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, c = lane & 15u, nblk = A.F / kBlock;
    const uint32_t n0 = 64u * blockIdx.x + 16u * (threadIdx.x >> 6);
    const uint32_t r = row0 + min(c, rows - 1u);
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    tile16(acc, ex.down_codes + (uint64_t)(n0 + c) * A.F + 32u * g,
           ex.down_scales + (uint64_t)(n0 / kBlock) * nblk, A.hq + (uint64_t)r * A.F + 32u * g,
           A.hs + (uint64_t)r * nblk, nblk);
    if (c >= rows) return;
    uint16_t *y = A.y + (uint64_t)A.route_index[r] * A.H + n0 + 4u * g;
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = f32_to_bf16(acc[i]);
}

struct Fp8Workspace {
    uint32_t *ids;
    float *weights;                /* the layer's routes */
    uint32_t *counts, *offsets, *unique, *summary, *token_index, *route_index;
    void *plan;
    size_t plan_bytes;
    uint32_t *tiles, *tile_count;
    uint32_t tile_cap;
    uint8_t *xq, *hq;
    float *xs, *hs, *h;
    uint16_t *y;
    void *router;
    size_t router_bytes, bytes;
};

Fp8Workspace carve(void *base, const k3_moe_shape &s, uint32_t T) {
    Fp8Workspace w{};
    uint8_t *p = (uint8_t *)base;
    size_t off = 0;
    auto take = [&](size_t n) {
        uint8_t *q = p ? p + off : nullptr;
        off += align256(n);
        return q;
    };
    const size_t routes = (size_t)T * s.top_k, E = s.expert_count;
    w.ids = (uint32_t *)take(4u * routes);
    w.weights = (float *)take(4u * routes);
    w.counts = (uint32_t *)take(4u * E);
    w.offsets = (uint32_t *)take(4u * (E + 1u));
    w.unique = (uint32_t *)take(4u * E);
    w.summary = (uint32_t *)take(16u);
    w.token_index = (uint32_t *)take(4u * routes);
    w.route_index = (uint32_t *)take(4u * routes);
    w.plan_bytes = k3_moe_plan_scratch_bytes(T, s.expert_count);
    w.plan = take(w.plan_bytes);
    w.tile_cap = (uint32_t)(routes / 16u + (E < routes ? E : routes));
    w.tiles = (uint32_t *)take(12u * (size_t)w.tile_cap);
    w.tile_count = (uint32_t *)take(4u);
    w.xq = take((size_t)T * s.hidden);
    w.xs = (float *)take((size_t)T * s.hidden / 32u);
    w.h = (float *)take(4u * routes * s.ffn);
    w.hq = take(routes * s.ffn);
    w.hs = (float *)take(routes * s.ffn / 32u);
    w.y = (uint16_t *)take(2u * routes * s.hidden);
    w.router_bytes = k3_moe_router_scratch_bytes(T, s.expert_count);
    w.router = take(w.router_bytes);
    w.bytes = off;
    return w;
}

bool fp8_shape_ok(const k3_moe_shape *s, uint32_t T) {
    return s && T != 0u && T <= 65535u && s->hidden != 0u && s->hidden % kBlock == 0u &&
           s->ffn != 0u && s->ffn % kBlock == 0u && s->expert_count != 0u &&
           s->expert_count <= 1024u && s->top_k != 0u && s->top_k <= 32u &&
           s->top_k <= s->expert_count && s->scaling_factor > 0.0f && s->activation <= 1u &&
           (s->activation == K3_MOE_ACT_SWIGLU || (s->beta > 0.0f && s->linear_beta > 0.0f));
}

bool launch_rows(uint8_t *codes, float *scales, const uint16_t *src, uint64_t blocks,
                 hipStream_t st) {
    hipLaunchKernelGGL(rows_kernel<uint16_t>, dim3((uint32_t)((blocks + 15u) / 16u)), dim3(256), 0,
                       st, codes, scales, src, blocks);
    return hipGetLastError() == hipSuccess;
}

/* The expert stage on routes in ws.ids (weights: wts). */
bool run_fp8_experts(const Fp8Workspace &ws, void *output, const void *hidden, const void *residual,
                     const float *wts, const k3_moe_fp8_expert *experts, const k3_moe_shape &s,
                     uint32_t T, hipStream_t st) {
    const uint32_t H = s.hidden, F = s.ffn, E = s.expert_count, k = s.top_k;
    if (!launch_rows(ws.xq, ws.xs, (const uint16_t *)hidden, (uint64_t)T * (H / kBlock), st) ||
        !k3_moe_route_plan(ws.counts, ws.offsets, ws.unique, ws.summary, ws.token_index,
                           ws.route_index, ws.ids, T, k, E, ws.plan, ws.plan_bytes, st))
        return false;
    hipLaunchKernelGGL(tiles_kernel, dim3(1), dim3(1024), 0, st, ws.tiles, ws.tile_count, ws.counts,
                       ws.offsets, E);
    const ExpertArgs A{experts, ws.tiles, ws.tile_count, ws.token_index, ws.route_index, ws.xq,
                       ws.xs, ws.h, ws.hq, ws.hs, ws.y, H, F, s.activation, s.beta, s.linear_beta};
    hipLaunchKernelGGL(gateup_kernel, dim3(F / 64u, ws.tile_cap), dim3(256), 0, st, A);
    const uint64_t blocks = (uint64_t)T * k * (F / kBlock);
    hipLaunchKernelGGL(rows_kernel<float>, dim3((uint32_t)((blocks + 15u) / 16u)), dim3(256), 0, st,
                       ws.hq, ws.hs, ws.h, blocks);
    hipLaunchKernelGGL(down_kernel, dim3(H / 64u, ws.tile_cap), dim3(256), 0, st, A);
    return hipGetLastError() == hipSuccess &&
           launch_combine(output, ws.y, residual, ws.ids, wts, T, H, k, E, st);
}

}  // namespace

size_t fp8_scratch_bytes(uint32_t T, uint32_t rows, uint32_t cols) {
    (void)rows;
    return align256((size_t)T * cols) + align256((size_t)T * (cols / kBlock) * 4u);
}

}  // namespace k3

using namespace k3;

extern "C" bool k3_moe_fp8_128_quantize_rows_bf16(uint8_t *codes, float *scales, const void *src,
                                                  uint32_t rows, uint32_t columns, void *stream) {
    const uint64_t blocks = (uint64_t)rows * (columns / kBlock);
    if (!codes || !scales || !src || rows == 0u || columns == 0u || columns % kBlock != 0u ||
        blocks > (1ull << 34) || ((uintptr_t)src % 16u) != 0u || ((uintptr_t)codes % 8u) != 0u ||
        ((uintptr_t)scales % 4u) != 0u)
        return false;
    return launch_rows(codes, scales, (const uint16_t *)src, blocks, (hipStream_t)stream);
}

extern "C" bool k3_moe_fp8_128_quantize_weight_bf16(uint8_t *codes, float *scales, const void *src,
                                                    uint32_t rows, uint32_t columns,
                                                    void *stream) {
    const uint64_t blocks = ((uint64_t)rows + kBlock - 1u) / kBlock * (columns / kBlock);
    if (!codes || !scales || !src || rows == 0u || columns == 0u || columns % kBlock != 0u ||
        blocks > 0x7fffffffull || ((uintptr_t)src % 16u) != 0u || ((uintptr_t)codes % 8u) != 0u ||
        ((uintptr_t)scales % 4u) != 0u)
        return false;
    hipLaunchKernelGGL(weight_kernel, dim3((uint32_t)blocks), dim3(256), 0, (hipStream_t)stream,
                       codes, scales, (const uint16_t *)src, rows, columns);
    return hipGetLastError() == hipSuccess;
}

extern "C" size_t k3_moe_fp8_128_scratch_bytes(uint32_t vector_count, uint32_t rows,
                                               uint32_t columns) {
    if (vector_count == 0u || vector_count > 65535u || rows == 0u || columns == 0u ||
        columns % kBlock != 0u)
        return 0u;
    return fp8_scratch_bytes(vector_count, rows, columns);
}

extern "C" bool k3_moe_fp8_128_gemm_bf16(void *output, const uint8_t *codes, const float *scales,
                                         const void *input, uint32_t vector_count, uint32_t rows,
                                         uint32_t columns, void *scratch, size_t scratch_bytes,
                                         void *stream) {
    if (!output || !codes || !scales || !input || vector_count == 0u || vector_count > 65535u ||
        rows == 0u || columns == 0u || columns % kBlock != 0u ||
        (((uintptr_t)codes | (uintptr_t)input) % 16u) != 0u || ((uintptr_t)scales % 4u) != 0u ||
        ((uintptr_t)output % 2u) != 0u)
        return false;
    const size_t need = fp8_scratch_bytes(vector_count, rows, columns);
    if (need != 0u && (!scratch || scratch_bytes < need || ((uintptr_t)scratch % 256u) != 0u))
        return false;
    const hipStream_t st = (hipStream_t)stream;
    uint8_t *xq = (uint8_t *)scratch;
    float *xs = (float *)(xq + align256((size_t)vector_count * columns));
    if (!launch_rows(xq, xs, (const uint16_t *)input, (uint64_t)vector_count * (columns / kBlock),
                     st))
        return false;
    hipLaunchKernelGGL(product_kernel, dim3((rows + 63u) / 64u, (vector_count + 15u) / 16u),
                       dim3(256), 0, st, (uint16_t *)output, codes, scales, xq, xs, vector_count,
                       rows, columns);
    return hipGetLastError() == hipSuccess;
}

extern "C" size_t k3_moe_fp8_workspace_bytes(const k3_moe_shape *shape, uint32_t token_count) {
    return fp8_shape_ok(shape, token_count) ? carve(nullptr, *shape, token_count).bytes : 0u;
}

namespace {

bool fp8_args_ok(const void *output, const void *hidden, const void *residual,
                 const k3_moe_fp8_expert *experts, const k3_moe_shape *shape, uint32_t T,
                 const void *workspace) {
    return output && hidden && experts && workspace && fp8_shape_ok(shape, T) &&
           (((uintptr_t)output | (uintptr_t)hidden | (uintptr_t)residual) % 16u) == 0u &&
           ((uintptr_t)workspace % 256u) == 0u;
}

}  // namespace

extern "C" bool k3_moe_fp8_experts_bf16(void *output, const void *hidden, const void *residual,
                                        const void *expert_ids, const void *expert_weights,
                                        const k3_moe_fp8_expert *experts,
                                        const k3_moe_shape *shape, uint32_t token_count,
                                        void *workspace, size_t workspace_bytes, void *stream) {
    if (!expert_ids || !expert_weights ||
        !fp8_args_ok(output, hidden, residual, experts, shape, token_count, workspace))
        return false;
    const Fp8Workspace ws = carve(workspace, *shape, token_count);
    if (workspace_bytes < ws.bytes) return false;
    const hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(routes_kernel, dim3((token_count + 255u) / 256u), dim3(256), 0, st, ws.ids,
                       (const uint32_t *)expert_ids, token_count, shape->top_k,
                       shape->expert_count);
    return hipGetLastError() == hipSuccess &&
           run_fp8_experts(ws, output, hidden, residual, (const float *)expert_weights, experts,
                           *shape, token_count, st);
}

extern "C" bool k3_moe_fp8_forward_bf16(void *output, const void *hidden, const void *residual,
                                        const void *router_weight, const void *router_bias,
                                        const k3_moe_fp8_expert *experts,
                                        const k3_moe_shape *shape, uint32_t token_count,
                                        void *expert_ids, void *expert_weights, void *workspace,
                                        size_t workspace_bytes, void *stream) {
    if (!router_weight || !router_bias || ((uintptr_t)router_weight % 16u) != 0u ||
        !fp8_args_ok(output, hidden, residual, experts, shape, token_count, workspace))
        return false;
    const Fp8Workspace ws = carve(workspace, *shape, token_count);
    if (workspace_bytes < ws.bytes) return false;
    const hipStream_t st = (hipStream_t)stream;
    const k3_moe_shape &s = *shape;
    const size_t route_bytes = (size_t)token_count * s.top_k * 4u;
    if (!k3_moe_router_bf16(ws.ids, ws.weights, hidden, router_weight, router_bias, token_count,
                            s.expert_count, s.hidden, s.top_k, s.scaling_factor, ws.router,
                            ws.router_bytes, st) ||
        (expert_ids && hipMemcpyAsync(expert_ids, ws.ids, route_bytes, hipMemcpyDefault, st) !=
                           hipSuccess) ||
        (expert_weights && hipMemcpyAsync(expert_weights, ws.weights, route_bytes,
                                          hipMemcpyDefault, st) != hipSuccess))
        return false;
    return run_fp8_experts(ws, output, hidden, residual, ws.weights, experts, s, token_count, st);
}
