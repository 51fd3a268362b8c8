/*
 * RMS norm with the residual's addition, to bf16 and to FP8-128 rows, and its
 * gradient. No reference counterpart as one call (the reference's engine adds,
 * then calls k3_rocm_rms_norm_bf16); the formulas are in include/k3_moe.h.
 *
 * A row is held by THREADS threads in CHUNKS pieces of eight values each, from
 * its one read to its writes: piece t + THREADS j is thread t's, so 16 lanes hold
 * the 128 values of an FP8-128 block. Rows of up to 2048 values go four to a block, a wave
 * each, without a barrier; longer ones take as many threads as leave two pieces to each, four past
 * 16384 values. Bound by memory: 8 bytes a value either way (residual in, sum out; both
 * gradients in), 7 with codes in place of the normed rows. us, rows x columns, forward and backward
 * (a large copy moves 5.2 TB/s): 32768 x 1024 44 and 51, 16384 x 2176 46 and 55, 8192 x 7168 83 (5.6
 * TB/s) and 97, of which the join of the weight's gradient 5; 4096 x 16384 95 and 107; 2048 x 32768
 * 106 and 142. With four pieces a thread 16384 x 2176 took 56 and 72, 8192 x 7168 88 and 98,
 * 4096 x 16384 105 and 204: fewer waves were under way, and of 1024 threads registers spilled.
 */
#include "k3_device.h"
#include "k3_fp8.h"
#include "k3_internal.h"
#include "../../include/k3_moe.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace k3 {
namespace {

constexpr uint32_t kMostColumns = 1u << 15, kMostRows = 65535u * 32u;

struct NormArgs {
    uint16_t *total, *normed; /* NULL: not wanted */
    uint8_t *codes;
    float *scales, *rstd;
    const uint16_t *x, *residual, *weight;
    uint32_t rows, cols;
    float eps;
};

__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
    return make_uint4(bf16_pack2(v[0], v[1]), bf16_pack2(v[2], v[3]), bf16_pack2(v[4], v[5]),
                      bf16_pack2(v[6], v[7]));
}

/* Sum over the THREADS threads of a row, the same order for each; red: its
 * THREADS / 64 floats in LDS (one wave: unused). */
template <uint32_t THREADS>
__device__ __forceinline__ float row_sum(float v, float *red) {
    v = wave_sum(v);
    if constexpr (THREADS > 64u) {
        if ((threadIdx.x & 63u) == 0u) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (uint32_t w = 1; w < THREADS / 64u; w++) v = __fadd_rn(v, red[w]);
    }
    return v;
}

template <uint32_t THREADS, int CHUNKS>
__global__ __launch_bounds__(THREADS < 256u ? 256u : THREADS) void norm_kernel(NormArgs A) {
    constexpr uint32_t ROWS = THREADS < 256u ? 256u / THREADS : 1u; /* of a block */
    __shared__ float red[THREADS / 64u];
    const uint32_t t = threadIdx.x % THREADS, pieces = A.cols / 8u;
    const uint32_t row = blockIdx.x * ROWS + threadIdx.x / THREADS;
    if (ROWS > 1u && row >= A.rows) return; /* a whole wave */
    const uint64_t at = (uint64_t)row * A.cols;
    uint4 xv[CHUNKS], rv[CHUNKS], wv[CHUNKS];
#pragma unroll
    for (int j = 0; j < CHUNKS; j++) {
        const uint32_t p = t + THREADS * (uint32_t)j;
        xv[j] = rv[j] = wv[j] = make_uint4(0u, 0u, 0u, 0u);
        if (p >= pieces) continue;
        xv[j] = ((const uint4 *)(A.x + at))[p];
        if (A.residual) rv[j] = ((const uint4 *)(A.residual + at))[p];
        wv[j] = ((const uint4 *)A.weight)[p];
    }
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < CHUNKS; j++) {
        const uint32_t p = t + THREADS * (uint32_t)j;
        float v[8], r[8];
        unpack8(xv[j], v);
        if (A.residual) { /* rounded: the sum is the next residual, and the gradient's input */
            unpack8(rv[j], r);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = __fadd_rn(v[i], r[i]);
            xv[j] = pack8(v);
            if (A.total && p < pieces) ((uint4 *)(A.total + at))[p] = xv[j];
            unpack8(xv[j], v);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) s = fmaf(v[i], v[i], s);
    }
    s = row_sum<THREADS>(s, red);
    const float rstd = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(s, (float)A.cols), A.eps)));
    if (A.rstd && t == 0u) A.rstd[row] = rstd;
#pragma unroll
    for (int j = 0; j < CHUNKS; j++) {
        const uint32_t p = t + THREADS * (uint32_t)j;
        float v[8], w[8];
        unpack8(xv[j], v);
        unpack8(wv[j], w);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = __fmul_rn(__fmul_rn(v[i], rstd), w[i]);
        if (A.normed && p < pieces) ((uint4 *)(A.normed + at))[p] = pack8(v);
        if (A.codes) { /* whole blocks of 16 lanes; of the fp32 values, rounded once */
            float scale, inv;
            fp8_scales(row_group_max<16>(max8(v)), scale, inv);
            if (p < pieces) {
                *(uint2 *)(A.codes + at + 8u * p) = fp8_codes8(v, inv);
                if ((p & 15u) == 0u) A.scales[(uint64_t)row * (pieces / 16u) + p / 16u] = scale;
            }
        }
    }
}

/*
 * Gradient. With n = s rstd weight (s the sum, d its gradient), dx = dtotal + rstd (d weight -
 * s rstd^2 mean(d weight s)) and dweight = sum over rows d s rstd. A block takes every
 * gridDim.x-th row (of its rows of a wave each, ROWS of them at once) and keeps the sums
 * of its columns in registers; they go to `parts`, a row for each block, and
 * norm_join_kernel adds those in their order. The sum's own gradient is loaded only behind the
 * sums' terms, under the wait for the row's sum: loaded with the others it took registers that cost
 * a wave (8192 x 7168 99.6 and 97.8 us).
 */
struct NormBackArgs {
    uint16_t *dx;
    float *parts; /* [blocks, cols] */
    const uint16_t *d, *total, *weight, *dtotal;
    const float *rstd;
    uint32_t rows, cols;
};

/* A row by offsets of 32 bits: pieces past its end, and all of no tensor, read as zeros and are not
 * written, without a branch; 64-bit addresses and the branches of a row's pieces took 60 registers. */
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_range(const void *base, uint64_t at, uint32_t cols) {
    return __builtin_amdgcn_make_buffer_rsrc((uint16_t *)base + at, 0, base ? (int)(2u * cols) : 0, 0x00027000);
}
__device__ __forceinline__ uint4 piece(__amdgpu_buffer_rsrc_t row, uint32_t p) {
    return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(row, (int)(16u * p), 0, 0));
}
__device__ __forceinline__ void put_piece(__amdgpu_buffer_rsrc_t row, uint32_t p, const uint4 &v) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, v), row, (int)(16u * p), 0, 0);
}
/* Unpacks of v from here on stay behind `behind`. */
__device__ __forceinline__ void keep_packed(uint4 &v, float &behind) {
    asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w), "+v"(behind));
}

template <uint32_t THREADS, int CHUNKS>
__global__ __launch_bounds__(THREADS < 256u ? 256u : THREADS) void norm_back_kernel(NormBackArgs A) {
    constexpr uint32_t ROWS = THREADS < 256u ? 256u / THREADS : 1u;
    __shared__ float red[2][THREADS / 64u];
    __shared__ float cols[ROWS > 1u ? ROWS : 1u][ROWS > 1u ? 8u * THREADS : 1u];
    const uint32_t t = threadIdx.x % THREADS, mine = threadIdx.x / THREADS, pieces = A.cols / 8u;
    const __amdgpu_buffer_rsrc_t weight = row_range(A.weight, 0u, A.cols);
    float sums[CHUNKS][8];
    uint4 wv[CHUNKS];
#pragma unroll
    for (int j = 0; j < CHUNKS; j++) {
        const uint32_t p = t + THREADS * (uint32_t)j;
        wv[j] = piece(weight, p);
#pragma unroll
        for (int i = 0; i < 8; i++) sums[j][i] = 0.0f;
    }
    uint32_t turn = 0u;
    for (uint32_t row = __builtin_amdgcn_readfirstlane(blockIdx.x * ROWS + mine); row < A.rows; row += gridDim.x * ROWS) {
        const uint64_t at = (uint64_t)row * A.cols;
        const __amdgpu_buffer_rsrc_t d_row = row_range(A.d, at, A.cols), s_row = row_range(A.total, at, A.cols),
                                     t_row = row_range(A.dtotal, at, A.cols), dx_row = row_range(A.dx, at, A.cols);
        uint4 dv[CHUNKS], sv[CHUNKS], tv[CHUNKS];
#pragma unroll
        for (int j = 0; j < CHUNKS; j++) {
            const uint32_t p = t + THREADS * (uint32_t)j;
            dv[j] = piece(d_row, p);
            sv[j] = piece(s_row, p);
        }
        const float rstd = A.rstd[row];
        float dot = 0.0f;
#pragma unroll
        for (int j = 0; j < CHUNKS; j++) {
            float d[8], s[8], w[8];
            keep_packed(dv[j], dot), keep_packed(sv[j], dot), keep_packed(wv[j], dot);
            unpack8(dv[j], d);
            unpack8(sv[j], s);
            unpack8(wv[j], w);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float ds = __fmul_rn(d[i], s[i]);
                dot = fmaf(ds, w[i], dot);
                sums[j][i] = fmaf(ds, rstd, sums[j][i]);
            }
        }
#pragma unroll
        for (int j = 0; j < CHUNKS; j++) {
            if (j == 0) asm volatile("" : "+v"(dot) : : "memory"); /* not ahead of the loop above */
            tv[j] = piece(t_row, t + THREADS * (uint32_t)j);
        }
        dot = row_sum<THREADS>(dot, red[turn & 1u]); /* two places: one barrier a row */
        turn++;
        /* unpacked anew below: kept over the sum, the floats would take twice the registers */
#pragma unroll
        for (int j = 0; j < CHUNKS; j++) {
            keep_packed(dv[j], dot), keep_packed(sv[j], dot), keep_packed(wv[j], dot);
        }
        const float back = __fmul_rn(__fmul_rn(rstd, rstd), __fdiv_rn(dot, (float)A.cols));
#pragma unroll
        for (int j = 0; j < CHUNKS; j++) {
            const uint32_t p = t + THREADS * (uint32_t)j;
            float d[8], s[8], w[8], b[8];
            unpack8(dv[j], d);
            unpack8(sv[j], s);
            unpack8(wv[j], w);
            unpack8(tv[j], b);
#pragma unroll
            for (int i = 0; i < 8; i++)
                d[i] = fmaf(rstd, fmaf(-s[i], back, __fmul_rn(d[i], w[i])), b[i]);
            put_piece(dx_row, p, pack8(d));
        }
    }
    float *part = A.parts + (uint64_t)blockIdx.x * A.cols;
    if constexpr (ROWS > 1u) { /* the block's rows of waves, in their order */
#pragma unroll
        for (int j = 0; j < CHUNKS; j++) {
            __syncthreads();
#pragma unroll
            for (uint32_t i = 0; i < 8u; i++) cols[mine][8u * t + i] = sums[j][i];
            __syncthreads();
            for (uint32_t c = threadIdx.x; c < 8u * THREADS; c += 256u) {
                float v = cols[0][c];
#pragma unroll
                for (uint32_t r = 1; r < ROWS; r++) v = __fadd_rn(v, cols[r][c]);
                const uint32_t col = 8u * THREADS * (uint32_t)j + c;
                if (col < A.cols) part[col] = v;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < CHUNKS; j++) {
            const uint32_t p = t + THREADS * (uint32_t)j;
            if (p >= pieces) continue;
            float4 *to = (float4 *)(part + 8u * p);
            to[0] = make_float4(sums[j][0], sums[j][1], sums[j][2], sums[j][3]);
            to[1] = make_float4(sums[j][4], sums[j][5], sums[j][6], sums[j][7]);
        }
    }
}

/* 32 columns a block, their parts in 32 runs (part q, q + 32, ...), then the runs. */
__global__ __launch_bounds__(1024) void norm_join_kernel(float *__restrict__ out, const float *__restrict__ parts,
                                                         uint32_t count, uint32_t cols) {
    __shared__ float runs[32][33];
    const uint32_t c = threadIdx.x & 31u, q = threadIdx.x >> 5, col = 32u * blockIdx.x + c;
    float v = 0.0f;
    if (col < cols) {
#pragma unroll 8
        for (uint32_t i = q; i < count; i += 32u) v = __fadd_rn(v, parts[(uint64_t)i * cols + col]);
    }
    runs[q][c] = v;
    __syncthreads();
    if (q != 0u || col >= cols) return;
    float sum = runs[0][c];
#pragma unroll
    for (int i = 1; i < 32; i++) sum = __fadd_rn(sum, runs[i][c]);
    out[col] = sum;
}

bool norm_sizes_ok(uint32_t rows, uint32_t cols) {
    return rows != 0u && rows <= kMostRows && cols != 0u && cols % 8u == 0u && cols <= kMostColumns;
}

/* Blocks of the gradient: each keeps a row of sums, so no more than the chip holds at once: three
 * a CU of up to 512 threads, one of 1024. */
uint32_t back_blocks(uint32_t rows, uint32_t cols) {
    const uint32_t groups = cols <= 2048u ? (rows + 3u) / 4u : rows;
    const uint32_t most = cols <= 8192u ? 768u : 256u;
    return groups < most ? groups : most;
}

}  // namespace
}  // namespace k3

using namespace k3;

extern "C" bool k3_moe_residual_norm_bf16(void *total, void *normed, uint8_t *codes, float *scales,
                                          float *rstd, const void *input, const void *residual,
                                          const void *weight, uint32_t rows, uint32_t columns,
                                          float epsilon, void *stream) {
    if (!input || !weight || !norm_sizes_ok(rows, columns) || (!normed && !codes && !total && !rstd) ||
        (residual != nullptr) != (total != nullptr) || (codes != nullptr) != (scales != nullptr) ||
        (codes && columns % kBlock != 0u) || !(epsilon >= 0.0f) ||
        (((uintptr_t)total | (uintptr_t)normed | (uintptr_t)input | (uintptr_t)residual | (uintptr_t)weight) %
         16u) != 0u ||
        (uintptr_t)codes % 8u != 0u || (((uintptr_t)scales | (uintptr_t)rstd) % 4u) != 0u)
        return false;
    /* a piece's place is read by the thread that writes there, so the sum and the normed
     * rows may each take an input's place */
    const uint64_t n = (uint64_t)rows * columns;
    const struct { const void *p; uint64_t bytes; } outs[] = {
        {total, 2u * n}, {normed, 2u * n}, {codes, n}, {scales, n / kBlock * 4u}, {rstd, 4u * (uint64_t)rows}};
    for (int i = 0; i < 5; i++) {
        if (!outs[i].p) continue;
        for (int j = i + 1; j < 5; j++)
            if (outs[j].p && overlap(outs[i].p, outs[i].bytes, outs[j].p, outs[j].bytes)) return false;
        for (const void *in : {input, residual})
            if (in && !(i < 2 && outs[i].p == in) && overlap(outs[i].p, outs[i].bytes, in, 2u * n))
                return false;
        if (overlap(outs[i].p, outs[i].bytes, weight, 2u * (uint64_t)columns)) return false;
    }
    const NormArgs A{(uint16_t *)total, (uint16_t *)normed, codes, scales, rstd, (const uint16_t *)input,
                     (const uint16_t *)residual, (const uint16_t *)weight, rows, columns, epsilon};
    const hipStream_t st = (hipStream_t)stream;
    const dim3 four((rows + 3u) / 4u), one(rows);
    if (columns <= 512u) hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_kernel<64u, 1>), four, dim3(256), 0, st, A);
    else if (columns <= 2048u) hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_kernel<64u, 4>), four, dim3(256), 0, st, A);
    else if (columns <= 4096u) hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_kernel<256u, 2>), one, dim3(256), 0, st, A);
    else if (columns <= 8192u) hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_kernel<512u, 2>), one, dim3(512), 0, st, A);
    else if (columns <= 16384u) hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_kernel<1024u, 2>), one, dim3(1024), 0, st, A);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_kernel<1024u, 4>), one, dim3(1024), 0, st, A);
    return hipGetLastError() == hipSuccess;
}

extern "C" size_t k3_moe_residual_norm_scratch_bytes(uint32_t rows, uint32_t columns) {
    if (!norm_sizes_ok(rows, columns)) return 0u;
    return 4u * (size_t)back_blocks(rows, columns) * columns;
}

extern "C" bool k3_moe_residual_norm_backward_bf16(void *input_gradient, float *weight_gradient,
                                                   const void *normed_gradient, const void *total,
                                                   const void *weight, const float *rstd,
                                                   const void *total_gradient, uint32_t rows,
                                                   uint32_t columns, void *scratch,
                                                   size_t scratch_bytes, void *stream) {
    if (!input_gradient || !weight_gradient || !normed_gradient || !total || !weight || !rstd || !scratch ||
        !norm_sizes_ok(rows, columns) || scratch_bytes < k3_moe_residual_norm_scratch_bytes(rows, columns) ||
        (((uintptr_t)input_gradient | (uintptr_t)normed_gradient | (uintptr_t)total | (uintptr_t)weight |
          (uintptr_t)total_gradient) % 16u) != 0u ||
        (((uintptr_t)weight_gradient | (uintptr_t)rstd) % 4u) != 0u || (uintptr_t)scratch % 256u != 0u)
        return false;
    const uint64_t n = 2u * (uint64_t)rows * columns;
    const uint64_t parts = k3_moe_residual_norm_scratch_bytes(rows, columns);
    const struct { const void *p; uint64_t bytes; } outs[] = {
        {input_gradient, n}, {weight_gradient, 4u * (uint64_t)columns}, {scratch, parts}};
    for (int i = 0; i < 3; i++) {
        for (int j = i + 1; j < 3; j++)
            if (overlap(outs[i].p, outs[i].bytes, outs[j].p, outs[j].bytes)) return false;
        for (const void *in : {normed_gradient, total, total_gradient})
            if (in && !(i == 0 && in == input_gradient) && overlap(outs[i].p, outs[i].bytes, in, n)) return false;
        if (overlap(outs[i].p, outs[i].bytes, weight, 2u * (uint64_t)columns) ||
            overlap(outs[i].p, outs[i].bytes, rstd, 4u * (uint64_t)rows))
            return false;
    }
    const NormBackArgs A{(uint16_t *)input_gradient, (float *)scratch, (const uint16_t *)normed_gradient,
                         (const uint16_t *)total, (const uint16_t *)weight, (const uint16_t *)total_gradient,
                         rstd, rows, columns};
    const hipStream_t st = (hipStream_t)stream;
    const uint32_t blocks = back_blocks(rows, columns);
    const dim3 grid(blocks);
    if (columns <= 512u) hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_back_kernel<64u, 1>), grid, dim3(256), 0, st, A);
    else if (columns <= 2048u) hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_back_kernel<64u, 4>), grid, dim3(256), 0, st, A);
    else if (columns <= 4096u) hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_back_kernel<256u, 2>), grid, dim3(256), 0, st, A);
    else if (columns <= 8192u) hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_back_kernel<512u, 2>), grid, dim3(512), 0, st, A);
    else if (columns <= 16384u) hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_back_kernel<1024u, 2>), grid, dim3(1024), 0, st, A);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(norm_back_kernel<1024u, 4>), grid, dim3(1024), 0, st, A);
    hipLaunchKernelGGL(norm_join_kernel, dim3((columns + 31u) / 32u), dim3(1024), 0, st, weight_gradient,
                       (const float *)scratch, blocks, columns);
    return hipGetLastError() == hipSuccess;
}
