/*
 * FP8-128: e4m3 codes with an fp32 scale for each block of 128 (128 values of
 * a token row, 128 x 128 of a weight), the product of such rows and weights,
 * and the routed experts on it. No reference counterpart; the encoding and the
 * products are defined in include/k3_moe.h.
 *
 *   rows_kernel           token rows
 *   weight_kernel         a weight, one 128 x 128 block a block
 *   product_one_kernel    few tokens' product
 *   product_tile_kernel   more tokens', tiles in LDS
 *   join_kernel           the parts of K of a product that was cut
 *   gateup_one_kernel     one token: act(gate . x, up . x) of its routes,
 *   down_one_kernel       their down products and weighted sum
 *   small_plan_kernel     up to 1024 tokens: their rows, and the experts' tiles
 *   tiles_kernel          the experts' tiles by k3_moe_route_plan's counts
 *   experts_tile_kernel   gate/up of all tiles; y[route] = bf16(down . h)
 *
 * MFMA operands (V_MFMA_F32_16X16X128_F8F6F4): lane 16 g + c holds 32 codes of
 * row c of the 16 x 128 slices: bytes [16 g, 16 g + 16) and [64 + 16 g, 64 +
 * 16 g + 16) of the row there, in every kernel alike, so an expert's sums have
 * the same bits in all of them. Weights are the first operand, tokens the
 * second: lane (g, c) of the result holds weight rows 4 g + i (i < 4) of token
 * c, so one factor scales all four.
 */
#include "k3_device.h"
#include "k3_fp8.h"
#include "k3_internal.h"
#include "k3_lds.h"
#include "../../include/k3_moe.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace k3 {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

/* A tile's 256 rows, and a batch's 65535, are addressed by 32 bits. */
constexpr uint32_t kMostAxis = 1u << 24, kMostWidth = 1u << 16;

inline size_t align256(size_t v) { return (v + 255u) & ~(size_t)255u; }
/* Scales of a row inside the library: whole groups of four. */
inline uint32_t scale_stride(uint32_t cols) { return (cols / kBlock + 3u) & ~3u; }

/* Sixteen lanes a block of 128 values, eight values a lane: one 16-byte load
 * (bf16), a maximum within a row of lanes, one 8-byte store. Scales: nblk of a
 * row, rows `stride` apart. Block q of the `blocks`, a row of lanes each. Bound by
 * memory: 8192 x 7168 in 30.8 us, 5.8 TB/s of bf16 read and codes written. */
struct RowArgs {
    uint8_t *codes;
    float *scales;
    const uint16_t *src;
    uint64_t blocks;
    uint32_t nblk, stride;
};
__device__ __forceinline__ void encode_block(const RowArgs &A, uint64_t q) {
    if (q >= A.blocks) return; /* whole rows of 16 lanes */
    const uint32_t l = threadIdx.x & 15u;
    const uint64_t at = kBlock * q + 8u * l;
    float v[8], scale, inv;
    load8(A.src + at, v);
    fp8_scales(row_group_max<16>(max8(v)), scale, inv);
    *(uint2 *)(A.codes + at) = fp8_codes8(v, inv);
    if (l != 0u) return;
    uint64_t to = q;
    if (A.stride != A.nblk) { /* a short division where it does */
        const uint64_t row = A.blocks >> 32 ? q / A.nblk : (uint32_t)q / A.nblk;
        to = q + row * (A.stride - A.nblk);
    }
    A.scales[to] = scale;
}
__global__ __launch_bounds__(256) void rows_kernel(RowArgs A) {
    encode_block(A, ((uint64_t)blockIdx.y * gridDim.x + blockIdx.x) * 16u + (threadIdx.x >> 4));
}

/* One block of 256 threads a 128 x 128 block: thread t holds eight columns of
 * rows t / 16 + 16 m; rows past the last are left out. The block stays in registers
 * between its maximum and its codes, so memory is read once: 4100 x 7168 in 15.3
 * us, 5.8 TB/s. */
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

/* The sums of a block's 128 code products. Not in fp32: of eight neighbours in a row the
 * instruction cuts each product, toward zero, to a multiple of 2^(E - 13), 2^E the power
 * of two of the largest, adds them up, and adds the sums of its 16 groups in fp32. A
 * block of random values is off by 2.0e-6 (rms) of the sum of its magnitudes, one of a
 * single sign comes out 2.5e-6 short, one whose terms span e^8 is off by up to 3e-4; fp32
 * in order is off by 2e-8. That is accepted for the rate: the codes themselves are within 2^-4
 * of their values, and the outputs' bf16 rounding is 1.7e-3 (4096 x 7168 x 7168: 1.2 %
 * of them a bf16 step off the rounded exact value, 0.1 % with fp32 sums). The 32-wide
 * instruction cuts the same; products of the same codes as bf16 are summed in fp32, at half
 * the rate. Tests: tests/test_gpu_fp8_sums.py. */
__device__ __forceinline__ f32x4 mfma_block(u32x4_t a0, u32x4_t a1, u32x4_t b0, u32x4_t b1) {
    const i32x8 a = {(int)a0.x, (int)a0.y, (int)a0.z, (int)a0.w,
                     (int)a1.x, (int)a1.y, (int)a1.z, (int)a1.w};
    const i32x8 b = {(int)b0.x, (int)b0.y, (int)b0.z, (int)b0.w,
                     (int)b1.x, (int)b1.y, (int)b1.z, (int)b1.w};
    /* no block scales: with constant zeros the unscaled form of the instruction
     * (alone on the part 4993 TFLOP/s, with scales of 2^0 4594) */
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 0,
                                                            0, 0, 0, 0, 0);
}

__device__ __forceinline__ uint2 bf16x4(const f32x4 &v) {
    return make_uint2(f32_to_bf16(v[0]) | (uint32_t)f32_to_bf16(v[1]) << 16,
                      f32_to_bf16(v[2]) | (uint32_t)f32_to_bf16(v[3]) << 16);
}
/* Columns n .. n + 3 of row t of a [T, N] output; wide: N % 4 == 0 and rows
 * 8-byte aligned. */
__device__ __forceinline__ void store_rows(uint16_t *out, const f32x4 &v, uint32_t t, uint32_t n,
                                           uint32_t T, uint32_t N, bool wide) {
    if (t >= T || n >= N) return;
    const uint2 u = bf16x4(v);
    uint16_t *p = out + (uint64_t)t * N + n;
    if (wide) {
        *(uint2 *)p = u;
        return;
    }
    p[0] = (uint16_t)u.x;
    if (n + 1u < N) p[1] = (uint16_t)(u.x >> 16);
    if (n + 2u < N) p[2] = (uint16_t)u.y;
    if (n + 3u < N) p[3] = (uint16_t)(u.y >> 16);
}

/* The activation and SiTU's constants: by = 1 / beta (at most the largest number,
 * so that 0 stays 0), by_linear = 1 / linear_beta. */
struct Activation {
    uint32_t kind;
    float beta, linear, by, by_linear;
};
Activation activation_of(const k3_moe_shape &s) {
    const auto inverse = [](float v) { return v < 0x1p-127f ? 0x1.fffffep127f : 1.0f / v; };
    return Activation{s.activation, s.beta, s.linear_beta, inverse(s.beta), inverse(s.linear_beta)};
}

/* In fp32: it is encoded in e4m3 next, and exp2 and the reciprocal of the hardware
 * (1 ulp), products with reciprocals and tanh_f32 are far inside that. SiTU costs
 * some 60 vector cycles a value: a division by each beta would be 30 more. */
__device__ __forceinline__ float act_f32(float g, float u, const Activation &A) {
    const float e = __builtin_amdgcn_exp2f(__fmul_rn(g, -1.44269504088896341f));
    const float s = __builtin_amdgcn_rcpf(__fadd_rn(1.0f, e));
    if (A.kind == K3_MOE_ACT_SWIGLU) return __fmul_rn(__fmul_rn(g, s), u);
    const float bg = __fmul_rn(A.beta, tanh_f32(__fmul_rn(g, A.by)));
    const float bu = __fmul_rn(A.linear, tanh_f32(__fmul_rn(u, A.by_linear)));
    return __fmul_rn(__fmul_rn(bg, s), bu);
}

/* ---------------------------------------------------------------------- */
/* one token                                                               */
/* ---------------------------------------------------------------------- */

/* A row of up to 64 scales by the lanes of a wave: loaded one at a time, each block
 * of columns would wait for its own. */
__device__ __forceinline__ float lane_scales(const float *row, uint32_t n) {
    return row[min(threadIdx.x & 63u, n - 1u)];
}
__device__ __forceinline__ float scale_at(float scales, uint32_t k) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(scales), (int)(k & 63u)));
}

/*
 * A wave's own ring of weights in LDS: M matrices x 16 rows x 128 columns a
 * stage. Direct-to-LDS loads take whole 128-byte lines (eight rows an
 * instruction); straight into the registers of the MFMA layout a load touches
 * 16 rows in 16-byte pieces, which holds a CU to about 10 bytes a clock (61
 * tokens' gate/up: 4.8 TB/s so, 6.1 TB/s through LDS). No wave waits for
 * another. Loads past the end take the last block again: the waits count them.
 */
template <int M, int R>
struct WaveRing {
    static constexpr uint32_t STAGE = 2048u * M, BYTES = STAGE * R;
    const uint8_t *src[M]; /* row 0 of the 16, at column 0 */
    uint32_t off[2];       /* this lane's place in the two loads of a matrix */
    uint8_t *smem;
    uint32_t base;

    __device__ __forceinline__ void init(uint8_t *lds, const uint8_t *const (&w)[M], uint32_t rows,
                                         uint32_t K) {
        const uint32_t L = threadIdx.x & 63u;
        smem = lds, base = lds_addr(lds);
#pragma unroll
        for (int m = 0; m < M; m++) src[m] = w[m];
#pragma unroll
        for (uint32_t h = 0; h < 2u; h++)
            off[h] = min(a_dma_row(L, h), rows - 1u) * K + 16u * a_dma_piece(L, h);
    }
    __device__ __forceinline__ void fetch(uint32_t block, uint32_t slot) const {
#pragma unroll
        for (int m = 0; m < M; m++)
#pragma unroll
            for (uint32_t h = 0; h < 2u; h++)
                dma<16>(src[m] + kBlock * block + off[h], smem + STAGE * slot + 2048u * m + 1024u * h);
    }
    /* The products of the stage in `slot` with the token codes at LDS address x. */
    __device__ __forceinline__ void products(f32x4 (&p)[M], uint32_t slot, uint32_t x) const {
        const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, c = lane & 15u;
        const uint32_t at = base + STAGE * slot;
        u32x4_t a[M][2], b[2];
        wait_vm<2 * M *(R - 1)>();
        asm volatile("" ::: "memory");
        static_for<M>([&](auto Q) {
            constexpr int m = decltype(Q)::value;
            a[m][0] = ds_read16<2048 * m>(at + a_slot(c, g));
            a[m][1] = ds_read16<2048 * m>(at + a_slot(c, 4u + g));
        });
        b[0] = ds_read16<0>(x + 16u * g);
        b[1] = ds_read16<64>(x + 16u * g);
        wait_lgkm<0>();
#pragma unroll
        for (int m = 0; m < M; m++) {
            after_wait(a[m][0]);
            after_wait(a[m][1]);
        }
        after_wait(b[0]);
        after_wait(b[1]);
#pragma unroll
        for (int m = 0; m < M; m++) p[m] = mfma_block(a[m][0], a[m][1], b[0], b[1]);
        asm volatile("" ::: "memory");
    }
};

__device__ __forceinline__ void ds_write8(uint32_t addr, uint2 v) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 w = {v.x, v.y};
    asm volatile("ds_write_b64 %0, %1" ::"v"(addr), "v"(w) : "memory");
}
__device__ __forceinline__ void ds_write4(uint32_t addr, uint32_t v) {
    asm volatile("ds_write_b32 %0, %1" ::"v"(addr), "v"(v) : "memory");
}
/* Between LDS writes and other waves' reads, with loads to LDS still out. */
__device__ __forceinline__ void lds_barrier() {
    wait_lgkm<0>();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

/* 16 lanes' part of an encoding: eight of a block's 128 values each, to codes and
 * (the first lane) its scale at LDS addresses. */
__device__ __forceinline__ void encode_lds(const float (&u)[8], uint32_t codes, uint32_t scale_at, bool first) {
    float scale, inv;
    fp8_scales(row_group_max<16>(max8(u)), scale, inv);
    ds_write8(codes, fp8_codes8(u, inv));
    if (first) ds_write4(scale_at, __float_as_uint(scale));
}

/* THREADS threads encode up to PER times as many pieces of eight values into LDS:
 * codes at `codes`, scales at `scales` (LDS addresses). Loads first, so that what
 * is issued between the two halves does not stand in their way. ENCODED: the tokens
 * come as codes with their scales and are copied. */
template <uint32_t THREADS, uint32_t PER, bool ENCODED = false>
struct TokenPart;
template <uint32_t THREADS, uint32_t PER>
struct TokenPart<THREADS, PER, true> {
    uint2 v[PER];
    float s[PER];
    __device__ __forceinline__ void load(const uint8_t *x, const float *scales, uint32_t n) {
#pragma unroll
        for (uint32_t i = 0; i < PER; i++) {
            const uint32_t q = min(threadIdx.x + THREADS * i, 16u * n - 1u);
            v[i] = ((const uint2 *)x)[q];
            s[i] = scales[q >> 4];
        }
    }
    __device__ __forceinline__ void encode(uint32_t n, uint32_t codes, uint32_t scales) const {
#pragma unroll
        for (uint32_t i = 0; i < PER; i++) {
            const uint32_t q = threadIdx.x + THREADS * i;
            if (q >= 16u * n) continue;
            ds_write8(codes + 8u * q, v[i]);
            if ((q & 15u) == 0u) ds_write4(scales + (q >> 2), __float_as_uint(s[i]));
        }
    }
};
template <uint32_t THREADS, uint32_t PER>
struct TokenPart<THREADS, PER, false> {
    uint4 v[PER];
    __device__ __forceinline__ void load(const uint16_t *x, uint32_t n) {
#pragma unroll
        for (uint32_t i = 0; i < PER; i++) /* past the end the last ones again */
            v[i] = ((const uint4 *)x)[min(threadIdx.x + THREADS * i, 16u * n - 1u)];
    }
    __device__ __forceinline__ void encode(uint32_t n, uint32_t codes, uint32_t scales) const {
#pragma unroll
        for (uint32_t i = 0; i < PER; i++) {
            const uint32_t q = threadIdx.x + THREADS * i;
            if (q >= 16u * n) continue; /* whole rows of 16 lanes */
            float u[8];
            unpack8(v[i], u);
            encode_lds(u, codes + 8u * q, scales + (q >> 2), (q & 15u) == 0u);
        }
    }
};

struct OneArgs {
    uint16_t *out;
    const uint8_t *codes;
    const float *scales;
    const uint16_t *x;      /* or, encoded, */
    const uint8_t *xq;
    const float *xs;
    uint32_t T, N, K;
};

/*
 * NT tokens (the last group's may be fewer) times a weight, 16 rows a block: its
 * eight waves take every eighth block of columns and add up through LDS in one
 * order. The tokens are encoded CHUNK blocks of columns at a time, by the block,
 * under the first weight loads; column c of the products is token min(c, NT - 1).
 * Each block encodes the tokens anew, which costs more the more blocks, tokens and
 * columns there are. us, here and by tiles with a launch for the codes and one for
 * the parts of K: 2048 x 7168, 1 token 5.7 and 12.4, 4 tokens 7.4 and 12.4, 8
 * tokens 9.8 and 12.4; 7168 x 7168 12.7, 17.5, 22.6 and 20.3 (one token's weights
 * at 4.1 TB/s and, of 2048 rows, 2.6: the first loads' latency is half of it); by 16
 * tokens, from a graph: 512 x 2048, 16 tokens 5.9 and 7.8, 128 tokens 6.4 and 8.4; 1024
 * x 4096, 64 tokens 8.6 and 9.4; 256 x 7168, 16 tokens 13.4 and 9.2.
 */
constexpr int kOneRing = 4;
inline bool one_launch(uint32_t T, uint32_t N, uint32_t K) {
    if (T <= 8u) return T <= 4u || N <= 4096u;
    return K <= 4096u && (T + 15ull) / 16u * ((N + 15u) / 16u) <= 256u;
}
template <uint32_t NT, uint32_t CHUNK, bool ENCODED> /* blocks of columns encoded at a time: 64 or 32 */
__global__ __launch_bounds__(512) void product_one_kernel(OneArgs P) {
    using Ring = WaveRing<1, kOneRing>;
    constexpr uint32_t TOKEN = CHUNK * (kBlock + 4u); /* codes, then scales */
    static_assert(CHUNK == 64u || CHUNK == 32u, "whole turns of the waves, whole loads");
    __shared__ __attribute__((aligned(1024))) uint8_t smem[8u * Ring::BYTES + NT * TOKEN];
    __shared__ float sums[8][NT][16];
    const uint32_t t0 = NT * blockIdx.y, T = min(NT, P.T - t0);
    const uint32_t lane = threadIdx.x & 63u, nblk = P.K / kBlock, n0 = 16u * blockIdx.x;
    const uint32_t c = lane & 15u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t codes = lds_addr(smem) + 8u * Ring::BYTES;
    const uint32_t mine = codes + TOKEN * min(c, NT - 1u);
    const float *ws = P.scales + (uint64_t)(n0 / kBlock) * nblk;
    /* lane q: the scale of the wave's q-th block of a chunk */
    float sw = ws[min(wave + 8u * (lane & 7u), nblk - 1u)];
    TokenPart<512u, CHUNK / 32u, ENCODED> x[NT];
    auto load = [&](uint32_t block, uint32_t n) {
#pragma unroll
        for (uint32_t t = 0; t < NT; t++) {
            const uint64_t row = t0 + min(t, T - 1u), at = row * P.K + kBlock * block;
            if constexpr (ENCODED) x[t].load(P.xq + at, P.xs + row * nblk + block, n);
            else x[t].load(P.x + at, n);
        }
    };
    load(0u, min(CHUNK, nblk));
    asm volatile("" ::: "memory"); /* issued before the weights, so that their waits leave those out */
    Ring ring;
    const uint8_t *const w[1] = {P.codes + (uint64_t)n0 * P.K};
    ring.init(smem + Ring::BYTES * wave, w, P.N - n0, P.K);
#pragma unroll
    for (uint32_t q = 0; q < kOneRing; q++) ring.fetch(min(wave + 8u * q, nblk - 1u), q);
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    uint32_t slot = 0u;
    for (uint32_t base = 0; base < nblk; base += CHUNK) {
        const uint32_t n = min(CHUNK, nblk - base);
        if (base != 0u) {
            sw = ws[min(base + wave + 8u * (lane & 7u), nblk - 1u)];
            load(base, n);
            lds_barrier(); /* the codes before have been read */
        }
#pragma unroll
        for (uint32_t t = 0; t < NT; t++) x[t].encode(n, codes + TOKEN * t, codes + TOKEN * t + CHUNK * kBlock);
        asm volatile("" : "+v"(sw)); /* waited for here, not in the loop */
        lds_barrier();
        for (uint32_t k = wave, q = 0; k < n; k += 8u, q++) {
            f32x4 p[1];
            uint32_t sx = ds_read4<CHUNK * kBlock>(mine + 4u * k);
            ring.products(p, slot, mine + kBlock * k); /* waits for sx too */
            after_wait(sx);
            const float f = __fmul_rn(__uint_as_float(sx), scale_at(sw, q));
#pragma unroll
            for (int r = 0; r < 4; r++) acc[r] = fmaf(p[0][r], f, acc[r]);
            ring.fetch(min(base + k + 8u * kOneRing, nblk - 1u), slot);
            slot = slot + 1u == (uint32_t)kOneRing ? 0u : slot + 1u;
        }
    }
    wait_vm<0>();
    if (c < NT)
#pragma unroll
        for (uint32_t r = 0; r < 4u; r++) sums[wave][c][4u * (lane >> 4) + r] = acc[r];
    __syncthreads();
    const uint32_t t = threadIdx.x >> 4, n = n0 + (threadIdx.x & 15u);
    if (t < T && n < P.N) {
        float v = 0.0f;
#pragma unroll
        for (int u = 0; u < 8; u++) v = __fadd_rn(v, sums[u][t][threadIdx.x & 15u]);
        P.out[(uint64_t)(t0 + t) * P.N + n] = f32_to_bf16(v);
    }
}

/* Route r of a token: its id, or E (none: from E on, or an earlier one's). All ids
 * come with one load. */
__device__ __forceinline__ uint32_t one_route(const uint32_t *ids, uint32_t r, uint32_t k, uint32_t E) {
    const uint32_t lane = threadIdx.x & 63u, id = lane < k ? ids[lane] : E;
    const uint32_t e = (uint32_t)__builtin_amdgcn_readlane((int)id, (int)r);
    return e >= E || __any(lane < r && id == e) ? E : e;
}

struct OneExpertArgs {
    const k3_moe_fp8_expert *experts;
    const uint32_t *ids;
    const float *weights;
    const uint16_t *x, *residual;
    uint16_t *out;
    float *h; /* [T k, F] */
    uint32_t H, F, E, k;
    Activation act;
};

/*
 * Gate and up of one route of a token, WAVES times 16 columns a block: 16 columns of
 * each a wave over the whole of K, RING blocks of 128 in flight. h is left in fp32,
 * so that a block need not hold the 128 columns of one of its scales and one
 * token's few columns reach every CU; the down kernel encodes it. LDS: the rings,
 * then the token's codes and scales. Bound by the weights (hidden 7168, ffn 2048, 8
 * experts: 41.8 us, 5.6 TB/s) and, of small layers, by the latency of the loads
 * (2048, 512, 4 experts: 6.6 us).
 */
constexpr uint32_t kOneHidden = 8192, kOneFfn = 4096; /* widths that a token's kernels hold in LDS */
template <uint32_t WAVES, int RING, uint32_t MOST> /* H at most */
__global__ __launch_bounds__(64 * WAVES) void gateup_one_kernel(OneExpertArgs A) {
    using Ring = WaveRing<2, RING>;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[WAVES * Ring::BYTES + MOST + MOST / 32u];
    const uint32_t cols = A.F / (16u * WAVES), r = blockIdx.x / cols, t = r / A.k;
    TokenPart<64u * WAVES, MOST / 8u / (64u * WAVES)> x;
    x.load(A.x + (uint64_t)t * A.H, A.H / kBlock);
    const uint32_t e = one_route(A.ids + t * A.k, r - t * A.k, A.k, A.E);
    if (e >= A.E) return;
    const k3_moe_fp8_expert ex = A.experts[e];
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, nblk = A.H / kBlock;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t f0 = 16u * (WAVES * (blockIdx.x % cols) + wave);
    const uint32_t codes = lds_addr(smem) + WAVES * Ring::BYTES, scales = codes + A.H;
    const uint64_t row = (uint64_t)(f0 / kBlock) * nblk;
    const float *gs = ex.gate_scales + row, *us = ex.up_scales + row;
    float sg = lane_scales(gs, nblk), su = lane_scales(us, nblk);
    asm volatile("" ::: "memory"); /* issued before the weights, so that their waits leave those out */
    Ring ring;
    const uint8_t *const w[2] = {ex.gate_codes + (uint64_t)f0 * A.H, ex.up_codes + (uint64_t)f0 * A.H};
    ring.init(smem + Ring::BYTES * wave, w, 16u, A.H);
#pragma unroll
    for (uint32_t q = 0; q < (uint32_t)RING; q++) ring.fetch(min(q, nblk - 1u), q);
    x.encode(nblk, codes, scales);
    asm volatile("" : "+v"(sg), "+v"(su)); /* waited for here, not in the loop */
    lds_barrier();
    f32x4 gate = {0.0f, 0.0f, 0.0f, 0.0f}, up = gate;
    uint32_t slot = 0u;
    for (uint32_t k = 0; k < nblk; k++) { /* nblk <= 64 */
        f32x4 p[2];
        uint32_t sx = ds_read4<0>(scales + 4u * k);
        ring.products(p, slot, codes + kBlock * k); /* waits for sx too */
        after_wait(sx);
        const float fg = __fmul_rn(__uint_as_float(sx), scale_at(sg, k));
        const float fu = __fmul_rn(__uint_as_float(sx), scale_at(su, k));
        ring.fetch(min(k + RING, nblk - 1u), slot);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            gate[i] = fmaf(p[0][i], fg, gate[i]);
            up[i] = fmaf(p[1][i], fu, up[i]);
        }
        slot = slot + 1u == (uint32_t)RING ? 0u : slot + 1u;
    }
    wait_vm<0>();
    if ((lane & 15u) != 0u) return;
    f32x4 h;
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = act_f32(gate[i], up[i], A.act);
    *(f32x4 *)(A.h + (uint64_t)r * A.F + f0 + 4u * g) = h;
}

/*
 * A token's output: 16 columns a block, a route a wave at a time (its activation
 * encoded into the wave's LDS under the first weight loads), then the weighted sum
 * in rank order and the residual (as the batch's combine). 22.5 us for 8 routes of
 * 7168 x 2048, 5.2 TB/s; 3.7 us for 4 of 2048 x 512.
 */
constexpr int kDownRing = 3;
template <uint32_t MOST> /* F at most: 2048 lets a CU hold two blocks */
__global__ __launch_bounds__(512) void down_one_kernel(OneExpertArgs A) {
    using Ring = WaveRing<1, kDownRing>;
    constexpr uint32_t kRow = MOST + 64u * (MOST / 2048u); /* codes and scales */
    __shared__ __attribute__((aligned(1024))) uint8_t smem[8u * (Ring::BYTES + kRow)];
    __shared__ float y[32][16];
    __shared__ uint32_t live[32];
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, nblk = A.F / kBlock;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n0 = 16u * blockIdx.x;
    uint8_t *mine = smem + (Ring::BYTES + kRow) * wave;
    const uint32_t codes = lds_addr(mine) + Ring::BYTES, scales = codes + MOST;
    const uint32_t r0 = blockIdx.y * A.k; /* the token's first route */
    for (uint32_t r = wave; r < A.k; r += 8u) {
        const uint32_t e = one_route(A.ids + r0, r, A.k, A.E);
        if (lane == 0u) live[r] = e < A.E;
        if (e >= A.E) continue;
        const k3_moe_fp8_expert ex = A.experts[e];
        const float *ws = ex.down_scales + (uint64_t)(n0 / kBlock) * nblk;
        float f = lane_scales(ws, nblk); /* nblk <= 64 */
        const f32x4 *h = (const f32x4 *)(A.h + (uint64_t)(r0 + r) * A.F);
        constexpr uint32_t PER = MOST / 512u;
        f32x4 v[PER][2];
#pragma unroll
        for (uint32_t i = 0; i < PER; i++) { /* past the end the last ones again */
            const uint32_t q = min(lane + 64u * i, A.F / 8u - 1u);
            v[i][0] = h[2u * q], v[i][1] = h[2u * q + 1u];
        }
        asm volatile("" ::: "memory"); /* issued before the weights, so that their wait leaves those out */
        Ring ring;
        const uint8_t *const w[1] = {ex.down_codes + (uint64_t)n0 * A.F};
        ring.init(mine, w, 16u, A.F);
#pragma unroll
        for (uint32_t q = 0; q < kDownRing; q++) ring.fetch(min(q, nblk - 1u), q);
#pragma unroll
        for (uint32_t i = 0; i < PER; i++) {
            const uint32_t q = lane + 64u * i;
            if (q >= A.F / 8u) continue; /* whole rows of 16 lanes */
            float u[8];
#pragma unroll
            for (int j = 0; j < 8; j++) u[j] = v[i][j >> 2][j & 3];
            encode_lds(u, codes + 8u * q, scales + (q >> 2), (q & 15u) == 0u);
        }
        /* a wave's LDS operations are in order */
        uint32_t sx = ds_read4<0>(scales + 4u * min(lane, nblk - 1u));
        wait_lgkm<0>();
        after_wait(sx);
        f = __fmul_rn(__uint_as_float(sx), f);
        asm volatile("" : "+v"(f)); /* waited for here, not in the loop */
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
        uint32_t slot = 0u;
        for (uint32_t k = 0; k < nblk; k++) {
            f32x4 p[1];
            ring.products(p, slot, codes + kBlock * k);
            ring.fetch(min(k + kDownRing, nblk - 1u), slot);
            const float s = scale_at(f, k);
#pragma unroll
            for (int i = 0; i < 4; i++) acc[i] = fmaf(p[0][i], s, acc[i]);
            slot = slot + 1u == (uint32_t)kDownRing ? 0u : slot + 1u;
        }
        wait_vm<0>(); /* before the wave's next route, or the block's end */
        if ((lane & 15u) == 0u)
#pragma unroll
            for (int i = 0; i < 4; i++) y[r][4u * g + i] = bf16_to_f32(f32_to_bf16(acc[i]));
    }
    __syncthreads();
    if (threadIdx.x >= 16u) return;
    float v = 0.0f;
    for (uint32_t r = 0; r < A.k; r++)
        if (live[r]) v = __fadd_rn(v, __fmul_rn(A.weights[r0 + r], y[r][threadIdx.x]));
    uint16_t o = f32_to_bf16(v);
    const uint64_t at = (uint64_t)blockIdx.y * A.H + n0 + threadIdx.x;
    if (A.residual) o = f32_to_bf16(__fadd_rn(bf16_to_f32(A.residual[at]), bf16_to_f32(o)));
    A.out[at] = o;
}

/* One of the `many` row tiles of an expert with n rows from `row` on: all that
 * a block needs to know comes with one read. */
struct ExpertTile {
    uint32_t row, n, index, many;
    k3_moe_fp8_expert ex;
};
/* Rows of each but the last of an expert's tiles: all of up to 128 rows in one, more
 * in as few tiles of at most 256 as hold them, of whole steps of 32 rows. The last has
 * what is left: of 1345 rows (six tiles) 65, of 1793 (eight) one. */
__device__ __forceinline__ uint32_t tile_height(uint32_t n) {
    const uint32_t steps = (n + 31u) / 32u, many = (n + 255u) / 256u;
    return n > 128u ? 32u * ((steps + many - 1u) / many) : n;
}

/* Tile classes by an expert's rows: up to 32, 64 and 128 (one tile), more (tiles of
 * up to 256 by tile_height). */
constexpr int kClasses = 4;

struct TileLists {
    ExpertTile *tiles[kClasses];
    uint32_t *count; /* [kClasses] */
};

/* ---------------------------------------------------------------------- */
/* tiles of many tokens                                                    */
/* ---------------------------------------------------------------------- */

/*
 * 64 WN weight rows x 32 TI tokens a block of 2 WN waves; wave (wn, wt) holds
 * weight rows 64 wn .. + 64 and the token subtiles (16 tokens) wt, wt + 2, ...:
 * a tile with fewer tokens costs its 32-token steps, evenly over the waves. A
 * stage is a block of 128 columns of both operands, in LDS through
 * direct-to-LDS loads (whole 128-byte lines, XOR-swizzled pieces), STAGES of
 * them in a ring. A wave keeps its four weight fragments of a stage in
 * registers and streams the token fragments: four MFMAs with C = 0 each, whose
 * result goes into the fp32 accumulator with one fma per value under the factor
 * sx sw, one subtile later. Token scales come four blocks at a time (16 bytes a
 * token) into two buffers; the weights' are held by the lanes of a wave, 64 blocks
 * at a time, and read out by index.
 *
 * 4096 tokens, 7168 x 7168: 206 us, 2.04 PFLOP/s; gate/up and down of 4096 tokens
 * (8 of 128 experts of 7168, 2048): 1.2 ms at 1.6 PFLOP/s and 0.72 ms at 1.34, with
 * 256 rows for every expert, so that none is cut in two, 1.09 and 0.65 ms. The part
 * holds its power there by its clock (1.75 to 2.0 GHz of 2.4): four fmas an MFMA on
 * random data run at 3.5 PFLOP/s without any load or LDS. Tiles of fewer stages (down
 * has 16) pay a block's start and its stores, some 5 us, more often.
 */
template <int WN_, int TI_, int STAGES_>
struct Tile {
    static constexpr int WN = WN_, TI = TI_, STAGES = STAGES_, WAVES = 2 * WN, THREADS = 64 * WAVES;
    static constexpr uint32_t BN = 64 * WN, BT = 32 * TI;
    static constexpr uint32_t A = BN * kBlock, B = BT * kBlock, STAGE = A + B;
    static constexpr uint32_t SROWS = BT < 64u ? 64u : BT, SBUF = 16u * SROWS;
    static constexpr uint32_t B_CHUNKS = 4 * TI; /* of 8 rows, 1 KB; fewer than the waves: some load the same */
    static constexpr int DA = 4, DB = B_CHUNKS < WAVES ? 1 : B_CHUNKS / WAVES, D = DA + DB; /* loads a wave */
    static constexpr uint32_t LDS = STAGES * STAGE + 2u * SBUF;
    static_assert(LDS <= 160u * 1024u, "LDS");
    static_assert(STAGES <= 5, "a buffer of scales is read for four stages, and the next but one comes after");
    /* Two stages: a stage's weights have been read once its first subtile is
     * under way, so after a second barrier in mid-stage their place takes the
     * weights of two stages on (they come from HBM, the tokens from the L2). */
    static constexpr bool EARLY = STAGES == 2;
    static __device__ __forceinline__ uint32_t b_chunk(uint32_t wave, uint32_t q) {
        return B_CHUNKS < WAVES ? wave % B_CHUNKS : DB * wave + q;
    }
};

enum TileMode { kDense, kGateUp, kDown };

struct TileArgs {
    /* dense: the weight; otherwise the experts and the tiles */
    const uint8_t *codes;
    const float *scales;
    TileLists lists;
    const uint32_t *token_index, *route_index;
    const uint8_t *xq; /* token rows, K wide */
    const float *xs;   /* their scales, rows xstride apart */
    uint32_t xstride;
    uint16_t *out;     /* dense [T, N]; down y [routes, N] */
    uint8_t *hq;       /* gate/up: activation rows, N = F wide */
    float *hs;
    uint32_t hstride;
    uint32_t T, N, K, tiles_n, tiles_t;
    uint32_t splits, span; /* dense: K in `splits` parts of `span` blocks (a multiple of 4) */
    f32x4 *part;           /* their sums, of more than one */
    Activation act;
    bool wide, wide16; /* the output takes 8-byte, 16-byte stores */
};

/* acc[j][i] += the product over all blocks, for the first TL token subtiles of a
 * wave (a loop of its own for each TL: a test inside it costs registers). */
template <class C>
struct TileRun {
    const uint8_t *a_base, *b_base; /* the sources of this wave's loads, and this lane's places */
    uint32_t a[C::DA], b[C::DB];
    const float *sx;                    /* of the scale loads, for waves that have one */
    bool has_sx;
    const float *sw0, *sw1;             /* weight scales of fragments 0, 1 and 2, 3 */
    uint32_t nblk, wave, lane, wn, wt;

    __device__ __forceinline__ void fetch_scales(uint8_t *smem, uint32_t s) const {
        if (has_sx && s % 4u == 0u && s < nblk)
            dma<16>((const uint8_t *)(sx + s),
                    smem + C::STAGES * C::STAGE + C::SBUF * ((s >> 2) & 1u) + 1024u * wave);
    }
    /* Load Q of stage s; past the end the last stage again, so that the counts
     * of the waits stay. */
    template <int Q>
    __device__ __forceinline__ void fetch_one(uint8_t *smem, uint32_t s, uint32_t slot) const {
        const uint32_t at = kBlock * (s < nblk ? s : nblk - 1u);
        uint8_t *st = smem + C::STAGE * slot;
        if constexpr (Q < C::DA)
            dma<16>(a_base + at + a[Q], st + 1024u * (C::DA * wave + Q));
        else
            dma<16>(b_base + at + b[Q - C::DA],
                    st + C::A + 1024u * C::b_chunk(wave, Q - C::DA));
    }
    template <int FROM, int TO>
    __device__ __forceinline__ void fetch(uint8_t *smem, uint32_t s, uint32_t slot) const {
        static_for<TO - FROM>([&](auto Q) { fetch_one<FROM + decltype(Q)::value>(smem, s, slot); });
    }

    static __device__ __forceinline__ void scale_in(f32x4 &acc, const f32x4 &p, float f) {
#pragma unroll
        for (int r = 0; r < 4; r++) acc[r] = fmaf(p[r], f, acc[r]);
    }

    /*
     * Step s of the loop, token subtile j: the reads of subtile j + 1, the wait
     * for those of j, four products. Before the last subtile's products the
     * stage's LDS has been read by this wave; behind a barrier there (all waves
     * have, and stage s + 1 has landed for all) its products run over the reads
     * of the next stage's first fragments, so that no step begins with an empty
     * matrix unit.
     */
    template <int TL, bool Two>
    __device__ __forceinline__ void run(f32x4 (&acc)[C::TI][4], uint8_t *smem) const {
        const uint32_t g = lane >> 4, c = lane & 15u;
        const uint32_t base = lds_addr(smem), lo = a_slot(c, g), hi = a_slot(c, 4u + g);
        const uint32_t a_at = base + 8192u * wn, b_at = base + C::A + 2048u * wt;
        const uint32_t s_at = base + C::STAGES * C::STAGE + 16u * (16u * wt + c);
        /* the weight scales of 64 blocks, in front of the loads whose waits they
         * would otherwise drain */
        float w0 = sw0[min(lane, nblk - 1u)], w1 = Two ? sw1[min(lane, nblk - 1u)] : 0.0f;
        asm volatile("" ::: "memory");
        f32x4 p[2][4]; /* the products of a subtile and of the one before, and their factors */
        float f[2][2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
        u32x4_t af[4][2], bf[2][2];
        uint32_t sx_[2];
        uint32_t st = 0u, sb = s_at; /* the stage's place, its scales' */
        auto read_a = [&](auto I) {
            constexpr int i = decltype(I)::value;
            af[i][0] = ds_read16<2048 * i>(a_at + st + lo);
            af[i][1] = ds_read16<2048 * i>(a_at + st + hi);
        };
        auto read_b = [&](auto J) {
            constexpr int j = decltype(J)::value;
            sx_[j & 1] = ds_read4<512 * j>(sb);
            bf[j & 1][0] = ds_read16<4096 * j>(b_at + st + lo);
            bf[j & 1][1] = ds_read16<4096 * j>(b_at + st + hi);
        };
        auto barrier = [] {
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < 4; i++) p[1][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < C::STAGES - 1; s++) {
            fetch_scales(smem, (uint32_t)s);
            fetch<0, C::D>(smem, (uint32_t)s, (uint32_t)s);
        }
        if constexpr (C::EARLY) fetch<0, C::DA>(smem, 1u, 1u);
        /* stage 0: what was issued after it may stay out */
        wait_vm<C::EARLY ? C::DA : C::D *(C::STAGES - 2)>();
        asm volatile("" : "+v"(w0), "+v"(w1));
        barrier();
        static_for<4>(read_a);
        read_b(std::integral_constant<int, 0>{});
        uint32_t slot = 0u, next = C::STAGES - 1;
        for (uint32_t s = 0; s < nblk; s++) {
            if (s % 64u == 0u && s != 0u) { /* of the next 64 blocks */
                const uint32_t q = s + lane < nblk ? s + lane : nblk - 1u;
                w0 = sw0[q];
                if (Two) w1 = sw1[q];
                /* waited for here: at its use the wait would drain the loads
                 * ahead in every stage */
                asm volatile("" : "+v"(w0), "+v"(w1));
            }
            const uint32_t ahead = s + C::STAGES - 1u, to = next;
            fetch_scales(smem, ahead);
            if constexpr (TL == 1) fetch<0, C::D>(smem, ahead, to);
            next = slot;
            slot = slot + 1u == (uint32_t)C::STAGES ? 0u : slot + 1u;
            const float sw_0 = scale_at(w0, s), sw_1 = Two ? scale_at(w1, s) : sw_0;
            static_for<TL>([&](auto J) {
                constexpr int j = decltype(J)::value;
                constexpr bool last = j + 1 == TL;
                if constexpr (!last) read_b(std::integral_constant<int, j + 1>{});
                wait_lgkm<last ? 0 : 3>(); /* the next subtile's reads stay out */
                if constexpr (j == 0) {
                    static_for<4>([&](auto I) {
                        after_wait(af[decltype(I)::value][0]);
                        after_wait(af[decltype(I)::value][1]);
                    });
                }
                after_wait(sx_[j & 1]);
                after_wait(bf[j & 1][0]);
                after_wait(bf[j & 1][1]);
                const float sx = __uint_as_float(sx_[j & 1]);
                f[j & 1][0] = __fmul_rn(sx, sw_0);
                f[j & 1][1] = Two ? __fmul_rn(sx, sw_1) : f[j & 1][0];
                if constexpr (last) {
                    /* this wave's loads of stage s + 1; later ones stay out */
                    wait_vm<C::EARLY ? C::DA : C::D *(C::STAGES - 2)>();
                    barrier();
                    st = C::STAGE * slot;
                    sb = s_at + C::SBUF * (((s + 1u) >> 2) & 1u) + 4u * ((s + 1u) & 3u);
                }
                /* a product, then the four fmas of the subtile before: they run
                 * while the matrix unit is busy */
                constexpr int q = (j + TL - 1) % TL;
                static_for<4>([&](auto I) {
                    constexpr int i = decltype(I)::value;
                    p[j & 1][i] = mfma_block(af[i][0], af[i][1], bf[j & 1][0], bf[j & 1][1]);
                    if constexpr (last) read_a(I);
                    scale_in(acc[q][i], p[(j + 1) & 1][i], f[(j + 1) & 1][i >> 1]);
                    __builtin_amdgcn_sched_barrier(0);
                    /* the loads ahead, spread over the products before the last
                     * subtile's: at once they would keep the waves from their reads */
                    constexpr int half = 4 * ((TL + 1) / 2), at = 4 * j + i;
                    if constexpr (TL == 1) {
                    } else if constexpr (C::EARLY) {
                        if constexpr (at == half - 1) barrier();
                        static_for<C::DB>([&](auto Q) {
                            if constexpr (decltype(Q)::value * (half - 1) / C::DB == at)
                                fetch_one<C::DA + decltype(Q)::value>(smem, ahead, to);
                        });
                        static_for<C::DA>([&](auto Q) {
                            if constexpr (half - 1 + decltype(Q)::value * (4 * (TL - 1) - half) / C::DA == at)
                                fetch_one<decltype(Q)::value>(smem, s + 2u, to ^ 1u);
                        });
                    } else {
                        static_for<C::D>([&](auto Q) {
                            if constexpr (decltype(Q)::value * half / C::D == at)
                                fetch_one<decltype(Q)::value>(smem, ahead, to);
                        });
                    }
                });
                if constexpr (last) read_b(std::integral_constant<int, 0>{});
            });
            if constexpr (TL % 2 != 0) { /* the next stage's first subtile has the same parity */
#pragma unroll
                for (int i = 0; i < 4; i++) p[1][i] = p[0][i];
                f[1][0] = f[0][0], f[1][1] = f[0][1];
            }
        }
        wait_lgkm<0>(); /* the reads past the end: their registers stay taken till here */
        static_for<4>([&](auto I) {
            after_wait(af[decltype(I)::value][0]);
            after_wait(af[decltype(I)::value][1]);
        });
        after_wait(sx_[0]);
        after_wait(bf[0][0]);
        after_wait(bf[0][1]);
#pragma unroll
        for (int i = 0; i < 4; i++) scale_in(acc[TL - 1][i], p[1][i], f[1][i >> 1]);
        wait_vm<0>(); /* the loads past the end land before the LDS is used again */
    }
};

/* Work L of `works` (blocks L, L + 8, ... lie on one XCD): XCD x takes a
 * contiguous range of them. Returns false past the end. */
__device__ __forceinline__ bool xcd_work(uint32_t L, uint32_t works, uint32_t &w) {
    const uint32_t per = (works + 7u) / 8u, j8 = L >> 3;
    w = (L & 7u) * per + j8;
    return j8 < per && w < works;
}

/* Work of `block` among `tiles` row tiles (list: the experts') x P.tiles_n column
 * blocks (dense: x parts of K). LDS: bytes of smem. */
template <class C, int MODE, uint32_t LDS>
__device__ __forceinline__ void tile_block(const TileArgs &P, uint8_t *smem, uint32_t block, uint32_t tiles,
                                           const ExpertTile *list) {
    static_assert(MODE != kGateUp || C::WN == 4, "a gate/up block holds whole scale blocks");
    TileRun<C> R;
    R.lane = threadIdx.x & 63u;
    R.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    R.wn = R.wave % C::WN, R.wt = R.wave / C::WN;
    const uint32_t L = R.lane, K = P.K, nblk = K / kBlock;
    uint32_t w;
    if (!xcd_work(block, tiles * P.tiles_n * (MODE == kDense ? P.splits : 1u), w)) return;
    const uint32_t split = MODE == kDense ? w % P.splits : 0u; /* a part of K */
    if constexpr (MODE == kDense) w /= P.splits;
    uint32_t row0, rows, col;
    const uint8_t *w0, *w1;
    if constexpr (MODE == kDense) { /* four token tiles at a time, down the weight's rows */
        const uint32_t grp = w / (4u * P.tiles_n), in = w % (4u * P.tiles_n);
        const uint32_t high = min(4u, tiles - 4u * grp);
        col = in / high;
        row0 = C::BT * (4u * grp + in % high), rows = min(C::BT, P.T - row0);
        w0 = w1 = P.codes;
        R.sw0 = R.sw1 = P.scales;
    } else {
        /* an expert's tiles of one column block are neighbours: they read the
         * same weights at about the same time, through the same L2 */
        const ExpertTile &t = list[w / P.tiles_n];
        const uint32_t local = t.index * P.tiles_n + w % P.tiles_n, height = tile_height(t.n);
        const uint32_t q = local % t.many;
        col = local / t.many;
        row0 = t.row + height * q, rows = min(height, t.n - height * q);
        w0 = MODE == kGateUp ? t.ex.gate_codes : t.ex.down_codes;
        w1 = t.ex.up_codes;
        R.sw0 = MODE == kGateUp ? t.ex.gate_scales : t.ex.down_scales;
        R.sw1 = MODE == kGateUp ? t.ex.up_scales : R.sw0;
    }
    const uint32_t n0 = (MODE == kGateUp ? 128u : C::BN) * col, nb0 = n0 / kBlock;
    {
        const uint32_t nb = MODE == kGateUp ? nb0 : min(nb0 + (R.wn >> 1), (P.N + kBlock - 1u) / kBlock - 1u);
        R.sw0 += (uint64_t)nb * nblk;
        R.sw1 += (uint64_t)nb * nblk;
    }
    const uint32_t k0 = MODE == kDense ? P.span * split : 0u; /* a multiple of 4 */
    R.nblk = MODE == kDense ? min(P.span, nblk - k0) : nblk;
    R.sw0 += k0, R.sw1 += k0;
    /* chunk q of A: rows 8 q .. + 8 of the tile; gate/up: wave wn's 64 rows are
     * 32 of gate, then the same 32 of up, so a loading wave has one of them */
    if constexpr (MODE == kGateUp)
        R.a_base = (R.wave & 1u ? w1 : w0) + (uint64_t)n0 * K;
    else
        R.a_base = w0 + (uint64_t)n0 * K + kBlock * k0;
    R.b_base = MODE == kGateUp ? P.xq : P.xq + (uint64_t)row0 * K + kBlock * k0;
#pragma unroll
    for (int q = 0; q < C::DA; q++) {
        const uint32_t ch = C::DA * R.wave + (uint32_t)q, h = ch & 1u;
        uint32_t r = 16u * (ch >> 1) + a_dma_row(L, h);
        if constexpr (MODE == kGateUp)
            r = 32u * (ch >> 3) + (r & 31u);
        else
            r = min(r, P.N - 1u - n0);
        R.a[q] = r * K + 16u * a_dma_piece(L, h);
    }
#pragma unroll
    for (int q = 0; q < C::DB; q++) {
        const uint32_t ch = C::b_chunk(R.wave, (uint32_t)q), h = ch & 1u;
        uint32_t r = min(16u * (ch >> 1) + a_dma_row(L, h), rows - 1u);
        if constexpr (MODE == kGateUp) r = P.token_index[row0 + r];
        R.b[q] = r * K + 16u * a_dma_piece(L, h);
    }
    {
        R.has_sx = 64u * R.wave < C::BT;
        uint32_t r = row0 + min(64u * R.wave + L, rows - 1u);
        if constexpr (MODE == kGateUp) r = P.token_index[r];
        R.sx = P.xs + (uint64_t)r * P.xstride + k0;
    }
    f32x4 acc[C::TI][4];
#pragma unroll
    for (int j = 0; j < C::TI; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[j][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    /* a loop for each number of 32-row steps from TI / 2 on: fewer steps (an expert's
     * last tile) take that one, with the last row in the place of those it has not */
    const uint32_t steps = (rows + 31u) / 32u;
    bool done = false;
    static_for<C::TI / 2>([&](auto Q) {
        constexpr int tl = C::TI / 2 + decltype(Q)::value;
        if (!done && steps <= (uint32_t)tl) {
            R.template run<tl, MODE == kGateUp>(acc, smem);
            done = true;
        }
    });
    if (!done) R.template run<C::TI, MODE == kGateUp>(acc, smem);
    const uint32_t g = L >> 4, c = L & 15u;
    if constexpr (MODE != kGateUp) {
        if (MODE == kDense && P.splits > 1u) { /* as they lie: join_kernel knows the layout */
            f32x4 *part = P.part + ((uint64_t)split * (tiles * P.tiles_n) + w) * (4u * C::TI * C::THREADS);
#pragma unroll
            for (int j = 0; j < C::TI; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) part[(4u * j + i) * C::THREADS + threadIdx.x] = acc[j][i];
        } else if (MODE == kDown || P.wide16) {
            /* the tile goes through LDS, 2 BN bytes a token, and leaves in
             * 16-byte pieces of whole rows; piece p of token r lies at p ^ r
             * modulo their number */
            constexpr uint32_t PIECES = C::BN / 8u;
            /* read here once: a load in the loop of stores would wait for each */
            static_assert(MODE != kDown || 2u * C::BN * C::BT + 4u * C::BT <= LDS, "tile and routes");
            uint32_t *const route = (uint32_t *)(smem + 2u * C::BN * C::BT);
            const uint32_t mine = MODE == kDown && threadIdx.x < rows ? P.route_index[row0 + threadIdx.x] : 0u;
            __syncthreads();
            static_for<C::TI>([&](auto J) {
                constexpr int j = decltype(J)::value;
                if (32u * j >= rows) return;
                const uint32_t r = 16u * (2u * j + R.wt) + c;
#pragma unroll
                for (uint32_t i = 0; i < 4u; i++) {
                    const uint32_t p = 8u * R.wn + 2u * i + (g >> 1);
                    *(uint2 *)(smem + 16u * (PIECES * r + (p ^ (r & (PIECES - 1u)))) + 8u * (g & 1u)) =
                        bf16x4(acc[j][i]);
                }
            });
            if (MODE == kDown && threadIdx.x < C::BT) route[threadIdx.x] = mine;
            __syncthreads();
            const uint32_t width = min(C::BN, P.N - n0); /* a multiple of 8 */
            const uint32_t p = threadIdx.x % PIECES;
            if (8u * p < width)
                for (uint32_t r = threadIdx.x / PIECES; r < rows; r += C::THREADS / PIECES) {
                    const uint32_t t = MODE == kDown ? route[r] : row0 + r;
                    *(uint4 *)(P.out + (uint64_t)t * P.N + n0 + 8u * p) =
                        *(const uint4 *)(smem + 16u * (PIECES * r + (p ^ (r & (PIECES - 1u)))));
                }
        } else {
            static_for<C::TI>([&](auto J) {
                constexpr int j = decltype(J)::value;
                const uint32_t r = 16u * (2u * j + R.wt) + c;
#pragma unroll
                for (uint32_t i = 0; i < 4u; i++)
                    store_rows(P.out, acc[j][i], row0 + r, n0 + 64u * R.wn + 16u * i + 4u * g, P.T, P.N,
                               P.wide);
            });
        }
    } else {
        /* the block's 128 columns are one scale block of each row: the maximum
         * over a wave's 32, then over its four neighbours' through LDS; codes
         * go through LDS too and leave as whole lines */
        __syncthreads();
        float *red = (float *)smem;             /* [4][BT] */
        uint8_t *rowbuf = smem + 16u * C::BT;   /* [BT][128] */
        static_for<C::TI>([&](auto J) {
            constexpr int j = decltype(J)::value;
            if (32u * j >= rows) return; /* tokens that the tile has not */
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float h = act_f32(acc[j][i][r], acc[j][i + 2][r], P.act);
                    acc[j][i][r] = h;
                    m = fmaxf(m, fabsf(h));
                }
            m = fmaxf(m, __shfl_xor(m, 16, 64));
            m = fmaxf(m, __shfl_xor(m, 32, 64));
            if (g == 0u) red[C::BT * R.wn + 16u * (2u * j + R.wt) + c] = m;
        });
        __syncthreads();
        static_for<C::TI>([&](auto J) {
            constexpr int j = decltype(J)::value;
            if (32u * j >= rows) return;
            const uint32_t r = 16u * (2u * j + R.wt) + c;
            float scale, inv;
            fp8_scales(fmaxf(fmaxf(red[r], red[C::BT + r]), fmaxf(red[2u * C::BT + r], red[3u * C::BT + r])),
                       scale, inv);
#pragma unroll
            for (uint32_t i = 0; i < 2u; i++) {
                const f32x4 h = acc[j][i];
                *(uint32_t *)(rowbuf + kBlock * r + 32u * R.wn + 16u * i + 4u * g) =
                    e4m3x2_raw<true>(__fmul_rn(h[2], inv), __fmul_rn(h[3], inv),
                                     e4m3x2_raw<false>(__fmul_rn(h[0], inv), __fmul_rn(h[1], inv), 0u));
            }
            if (R.wn == 0u && g == 0u && r < rows) P.hs[(uint64_t)(row0 + r) * P.hstride + nb0] = scale;
        });
        __syncthreads();
        for (uint32_t q = threadIdx.x; q < 8u * rows; q += 512u)
            *(uint4 *)(P.hq + (uint64_t)(row0 + (q >> 3)) * P.N + n0 + 16u * (q & 7u)) =
                *(const uint4 *)(rowbuf + 16u * q);
    }
}

template <class C>
__global__ __launch_bounds__(C::THREADS, 2) void product_tile_kernel(TileArgs P) {
    __shared__ __attribute__((aligned(1024))) uint8_t smem[C::LDS];
    tile_block<C, kDense, C::LDS>(P, smem, blockIdx.x, P.tiles_t, nullptr);
}

using Tile32 = Tile<4, 1, 4>;
using Tile64 = Tile<4, 2, 3>;
using Tile128 = Tile<4, 4, 3>;
using Tile256 = Tile<4, 8, 2>;
/* half as many rows: few tokens' products */
using Half32 = Tile<2, 1, 3>;
using Half64 = Tile<2, 2, 3>;
using Half128 = Tile<2, 4, 2>;

/* All tiles of the experts' gate/up, or down, in one launch: the classes one
 * behind the other, the largest tiles first, each on whole groups of eight
 * blocks. A CU holds one block of any class, so the largest's registers and LDS
 * cost the others nothing (a launch for each class took 3 to 5 us where it had no
 * tile). */
template <int MODE>
__global__ __launch_bounds__(512, 2) void experts_tile_kernel(TileArgs P) {
    __shared__ __attribute__((aligned(1024))) uint8_t smem[Tile128::LDS];
    static_assert(Tile128::LDS >= Tile256::LDS && Tile128::LDS >= Tile64::LDS &&
                  Tile128::LDS >= Tile32::LDS, "LDS of every class");
    const uint4 count = *(const uint4 *)P.lists.count;
    const uint32_t n[kClasses] = {count.x, count.y, count.z, count.w};
    uint32_t b = blockIdx.x, cls = kClasses;
#pragma unroll
    for (int q = kClasses - 1; q >= 0; q--) {
        const uint32_t blocks = 8u * ((n[q] * P.tiles_n + 7u) / 8u);
        if (cls != (uint32_t)kClasses) continue;
        if (b < blocks) cls = (uint32_t)q;
        else b -= blocks;
    }
    switch (cls) {
    case 0: tile_block<Tile32, MODE, sizeof smem>(P, smem, b, n[0], P.lists.tiles[0]); break;
    case 1: tile_block<Tile64, MODE, sizeof smem>(P, smem, b, n[1], P.lists.tiles[1]); break;
    case 2: tile_block<Tile128, MODE, sizeof smem>(P, smem, b, n[2], P.lists.tiles[2]); break;
    case 3: tile_block<Tile256, MODE, sizeof smem>(P, smem, b, n[3], P.lists.tiles[3]); break;
    }
}

/* Output of a product whose K was split: the parts in their order. A block adds
 * one accumulator (token subtile j, fragment i) of every wave of a tile, so that
 * all CUs read: 4.2 us for 37 tokens of 7168 x 7168 in four parts (the last block of
 * a tile alone would read its 128 KB in 5 us). */
template <class C>
__global__ __launch_bounds__(C::THREADS) void join_kernel(TileArgs P) {
    const uint32_t w = blockIdx.x / (4u * C::TI), ji = blockIdx.x % (4u * C::TI);
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, wn = wave % C::WN, wt = wave / C::WN;
    const uint32_t grp = w / (4u * P.tiles_n), in = w % (4u * P.tiles_n);
    const uint32_t high = min(4u, P.tiles_t - 4u * grp);
    const uint32_t t = C::BT * (4u * grp + in % high) + 16u * (2u * (ji >> 2) + wt) + (lane & 15u);
    const uint32_t n = C::BN * (in / high) + 64u * wn + 16u * (ji & 3u) + 4u * (lane >> 4);
    if (t >= P.T || n >= P.N) return;
    const uint64_t works = P.tiles_t * P.tiles_n, stride = works * (4u * C::TI * C::THREADS);
    const f32x4 *part = P.part + ((uint64_t)w * (4u * C::TI) + ji) * C::THREADS + threadIdx.x;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (uint32_t z = 0; z < P.splits; z++) {
        const f32x4 p = part[stride * z];
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] = __fadd_rn(v[r], p[r]);
    }
    store_rows(P.out, v, t, n, P.T, P.N, P.wide);
}

/* ---------------------------------------------------------------------- */
/* routes and tiles of the experts                                         */
/* ---------------------------------------------------------------------- */

typedef uint32_t u32x4_8 __attribute__((ext_vector_type(4), aligned(8))); /* two addresses */

/* By a block of 1024 threads, thread e with expert e's n rows and descriptor (ex):
 * each class's tiles in expert order. `row` is the expert's first row; FIRST: it is
 * the sum of the earlier experts' n, and set here. The four classes' tiles are
 * counted in 16 bits each of one word (65535 tokens of 32 routes are 9215 tiles at
 * most). */
template <bool FIRST>
__device__ __forceinline__ void list_tiles(const TileLists &Q, uint32_t &row, uint32_t n,
                                           u32x4_8 ex0, u32x4_8 ex1, u32x4_8 ex2) {
    static_assert(sizeof(ExpertTile) == 64 && sizeof(k3_moe_fp8_expert) == 48, "four stores");
    static_assert(kClasses == 4, "16 bits each");
    __shared__ unsigned long long tiles_of[16];
    __shared__ uint32_t rows_of[16];
    const uint32_t e = threadIdx.x, lane = e & 63u, wave = e >> 6;
    const uint32_t cls = n <= 32u ? 0u : n <= 64u ? 1u : n <= 128u ? 2u : 3u;
    const uint32_t height = n ? tile_height(n) : 1u, many = (n + height - 1u) / height;
    unsigned long long inc = (unsigned long long)many << (16u * cls);
    uint32_t rows = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned long long a = __shfl_up(inc, o, 64);
        const uint32_t r = FIRST ? __shfl_up(rows, o, 64) : 0u;
        if ((int)lane >= o) inc += a, rows += r;
    }
    if (lane == 63u) tiles_of[wave] = inc, rows_of[wave] = rows;
    __syncthreads();
    unsigned long long at = inc - ((unsigned long long)many << (16u * cls)), total = 0ull;
    if (FIRST) row = rows - n;
#pragma unroll
    for (uint32_t w = 0; w < 16u; w++) {
        if (w < wave) {
            at += tiles_of[w];
            if (FIRST) row += rows_of[w];
        }
        total += tiles_of[w];
    }
    const uint32_t to = (uint32_t)(at >> (16u * cls)) & 0xffffu;
    ExpertTile *const low = cls & 1u ? Q.tiles[1] : Q.tiles[0];
    ExpertTile *const high = cls & 1u ? Q.tiles[3] : Q.tiles[2];
    ExpertTile *const list = cls & 2u ? high : low;
    for (uint32_t i = 0; i < many; i++) {
        u32x4_8 *const t = (u32x4_8 *)(list + to + i);
        t[0] = u32x4_8{row, n, i, many};
        t[1] = ex0, t[2] = ex1, t[3] = ex2;
    }
    if (e == 0u) {
#pragma unroll
        for (int q = 0; q < kClasses; q++) Q.count[q] = (uint32_t)(total >> (16 * q)) & 0xffffu;
    }
}

/* By the plan's counts and first rows, in block 0; the others encode the tokens'
 * rows meanwhile. */
__global__ __launch_bounds__(1024) void tiles_kernel(TileLists Q, const uint32_t *__restrict__ counts,
                                                     const uint32_t *__restrict__ offsets,
                                                     const k3_moe_fp8_expert *__restrict__ experts,
                                                     uint32_t E, RowArgs R) {
    if (blockIdx.x != 0u) {
        encode_block(R, (blockIdx.x - 1u) * 64u + (threadIdx.x >> 4));
        return;
    }
    const uint32_t e = threadIdx.x;
    const u32x4_8 *const ex = (const u32x4_8 *)(experts + min(e, E - 1u));
    uint32_t row = offsets[min(e, E - 1u)];
    list_tiles<false>(Q, row, e < E ? counts[e] : 0u, ex[0], ex[1], ex[2]);
}

/* Up to 1024 tokens: the plan (k3_moe_route_plan's order) and the tiles as block
 * 0's work, while the others encode the tokens' rows: five launches in one. Thread
 * t < T of block 0 holds token t's routes; an expert's rows are the set bits of
 * its masks, a word for each 64 tokens: WORDS of them at most. 7.5 us for 61 tokens of
 * 8 routes (three barriers, the ids' and descriptors' latency, two scans); six
 * launches took 23 us. */
constexpr uint32_t kSmallPlan = 1024, kFewWords = 4096, kMostWords = 16384;
struct PlanArgs {
    TileLists lists;
    uint32_t *token_index, *route_index;
    const uint32_t *ids;
    const k3_moe_fp8_expert *experts;
    uint32_t T, k, E;
    RowArgs rows;
};
template <int K, uint32_t WORDS>
__global__ __launch_bounds__(1024) void small_plan_kernel(PlanArgs A) {
    __shared__ unsigned long long masks[WORDS]; /* [waves][E] */
    __shared__ uint32_t first[1024];
    if (blockIdx.x != 0u) {
        encode_block(A.rows, (blockIdx.x - 1u) * 64u + (threadIdx.x >> 4));
        return;
    }
    const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6, waves = (A.T + 63u) / 64u;
    const u32x4_8 *const ex = (const u32x4_8 *)(A.experts + min(t, A.E - 1u));
    const u32x4_8 ex0 = ex[0], ex1 = ex[1], ex2 = ex[2];
    asm volatile("" ::: "memory"); /* issued here, before the routes are waited for */
    uint32_t e[K];
    if (t < A.T) token_routes<K>(A.ids, t, A.k, A.E, e);
    for (uint32_t i = t; i < waves * A.E; i += 1024u) masks[i] = 0ull;
    __syncthreads();
    if (t < A.T) {
#pragma unroll
        for (int r = 0; r < K; r++)
            if (e[r] < A.E) atomicOr(&masks[wave * A.E + e[r]], 1ull << lane);
    }
    __syncthreads();
    uint32_t n = 0u, row = 0u;
    if (t < A.E)
        for (uint32_t w = 0; w < waves; w++) n += (uint32_t)__popcll(masks[w * A.E + t]);
    list_tiles<true>(A.lists, row, n, ex0, ex1, ex2);
    first[t] = row;
    __syncthreads();
    if (t >= A.T) return;
#pragma unroll
    for (int r = 0; r < K; r++) {
        if (e[r] >= A.E) continue;
        uint32_t at = first[e[r]] + (uint32_t)__popcll(masks[wave * A.E + e[r]] & ((1ull << lane) - 1ull));
        for (uint32_t w = 0; w < wave; w++) at += (uint32_t)__popcll(masks[w * A.E + e[r]]);
        A.token_index[at] = t;
        A.route_index[at] = t * A.k + (uint32_t)r;
    }
}

/* Whether a few tokens go through the experts one by one, in two launches. Tiles
 * take four and read an expert once however many tokens chose it: 14 us or some
 * 64 MB of weights read again, by the number of experts that T tokens choose if
 * each chooses at random. (us, one by one and by tiles; hidden 2048, ffn 512, 4 of 64
 * experts: 2 tokens 11.1 and 26.1, 8 tokens 22.4 and 32.1; 7168, 2048, 8 of 128:
 * 2 tokens 126 and 134, 4 tokens level, 8 tokens 451 and 413.) */
constexpr uint32_t kOneTokensMost = 64;
bool one_by_one(uint32_t T, const k3_moe_shape &s) {
    if (T > kOneTokensMost || s.hidden > kOneHidden || s.ffn > kOneFfn) return false;
    double miss = 1.0; /* of an expert by all tokens */
    for (uint32_t t = 0; t < T; t++) miss *= 1.0 - (double)s.top_k / s.expert_count;
    const double again = (double)T * s.top_k - s.expert_count * (1.0 - miss);
    return T == 1u || again * 3.0 * s.hidden * s.ffn < 64e6;
}

struct Fp8Workspace {
    uint32_t *ids;
    float *weights;                /* the layer's routes */
    uint32_t *counts, *offsets, *unique, *summary, *token_index, *route_index;
    void *plan;
    size_t plan_bytes;
    TileLists lists;
    uint32_t tile_cap; /* most tiles of all classes */
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
    /* an expert has a token's route at most once: T rows at most; n rows are
     * cut into at most 1 + n / 256 tiles, of the last class into at most n / 128 */
    static constexpr size_t least[kClasses] = {1u, 33u, 65u, 128u};
    const size_t used = E < routes ? E : routes;
    for (int q = 0; q < kClasses; q++) {
        const size_t n = T < least[q] ? 0u : routes / least[q];
        w.lists.tiles[q] = (ExpertTile *)take(sizeof(ExpertTile) * (q < 3 && n > E ? E : n));
    }
    w.tile_cap = (uint32_t)(used + routes / 256u);
    w.lists.count = (uint32_t *)take(4u * kClasses);
    w.xq = take((size_t)T * s.hidden);
    w.xs = (float *)take(4u * (size_t)T * scale_stride(s.hidden));
    const size_t from = off;
    w.hq = take(routes * s.ffn);
    w.hs = (float *)take(4u * routes * scale_stride(s.ffn));
    w.y = (uint16_t *)take(2u * routes * s.hidden);
    /* tokens that go one by one need h instead; room for it whenever fewer tokens
     * might, so that a workspace sized for more tokens serves them */
    w.h = (float *)w.hq;
    const size_t few = align256(4u * (size_t)(T < kOneTokensMost ? T : kOneTokensMost) * s.top_k * s.ffn);
    if (s.hidden <= kOneHidden && s.ffn <= kOneFfn && off < from + few) off = from + few;
    w.router_bytes = router_scratch_up_to(T, s.expert_count);
    w.router = take(w.router_bytes);
    w.bytes = off;
    return w;
}

bool fp8_shape_ok(const k3_moe_shape *s, uint32_t T) {
    return s && T != 0u && T <= 65535u && s->hidden != 0u && s->hidden % kBlock == 0u &&
           s->hidden <= kMostWidth && s->ffn != 0u && s->ffn % kBlock == 0u &&
           s->ffn <= kMostWidth && s->expert_count != 0u &&
           s->expert_count <= 1024u && s->top_k != 0u && s->top_k <= 32u &&
           s->top_k <= s->expert_count && s->scaling_factor > 0.0f && s->activation <= 1u &&
           (s->activation == K3_MOE_ACT_SWIGLU || (s->beta > 0.0f && s->linear_beta > 0.0f));
}

/* Rows of `cols` bf16 values to encode; scales of a row `stride` apart. */
constexpr uint64_t kMostGrid = 1u << 20; /* a launch's x axis is under 2^32 threads */
RowArgs row_args(uint8_t *codes, float *scales, const void *src, uint32_t rows, uint32_t cols,
                 uint32_t stride) {
    return RowArgs{codes, scales, (const uint16_t *)src, (uint64_t)rows * (cols / kBlock), cols / kBlock,
                   stride};
}
bool launch_rows(const RowArgs &A, hipStream_t st) {
    const uint64_t n = (A.blocks + 15u) / 16u;
    const uint32_t x = (uint32_t)(n < kMostGrid ? n : kMostGrid);
    hipLaunchKernelGGL(rows_kernel, dim3(x, (uint32_t)((n + x - 1u) / x)), dim3(256), 0, st, A);
    return hipGetLastError() == hipSuccess;
}

/* Scales [T, nblk] as rows `stride` apart, which tiles read four at a time. */
__global__ __launch_bounds__(256) void spread_scales_kernel(float *__restrict__ to,
                                                            const float *__restrict__ from, uint32_t T,
                                                            uint32_t nblk, uint32_t stride) {
    const uint64_t n = (uint64_t)T * stride;
    for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < n; i += 256ull * gridDim.x) {
        const uint64_t t = i / stride, b = i % stride;
        to[i] = b < nblk ? from[t * nblk + b] : 0.0f;
    }
}

/* How a product of more tokens is cut: its tile, and K in `splits` parts of `span`
 * blocks. */
struct Cut {
    int tile; /* 0 .. 4: Half32, Half64, Half128, Tile128, Tile256 */
    uint32_t tiles_t, tiles_n, splits, span;
};

/* Memory for the parts of K, which no cut exceeds: up to 16 parts, 768 blocks, and
 * tiles of 32, 64 or 128 rows for up to as many tokens (the cost rule alone picks
 * nothing larger: replayed for 6.5 million sizes up to 7424 x 8192, 4200 tokens, and
 * 20 million up to the limits). It grows with the tokens only, so that scratch sized
 * for more of them serves fewer. 7168 x 7168: 12 MiB up to 32 tokens, 32 from 65 on. */
constexpr size_t kMostParts = 32u << 20;
constexpr uint32_t kMostSplits = 16, kMostCutBlocks = 768;
size_t parts_room(uint32_t T, uint32_t N, uint32_t K) {
    const uint64_t groups = (K / kBlock + 3u) / 4u, splits = groups < kMostSplits ? groups : kMostSplits;
    if (splits < 2u) return 0u;
    const uint64_t height = T <= 32u ? 32u : T <= 64u ? 64u : T <= 128u ? 128u : (T + 255ull) / 256u * 256u;
    const uint64_t width = (N + 255ull) / 256u * 256u * splits, cut = 128u * kMostCutBlocks;
    const uint64_t most = 4u * height * (width < cut ? width : cut);
    return most < kMostParts ? most : kMostParts;
}

/*
 * The cheapest of all cuts, by what tiles cost on the part: nanoseconds of a
 * stage (128 columns) of a block that has a CU to itself, and a block's share
 * with several (tiles of 128 rows lie two a CU); a part of K in memory at 5
 * TB/s, written and read, and 3 us for the launch that adds them. (us, 2048 x
 * 7168, the tiles of 128 x 64, 128 x 128, 256 x 128 and 256 x 256: 512 tokens 25.1,
 * 26.5, 26.3, 34.3; 1024 tokens 35.2, 37.9, 39.4, 43.6; 4096 tokens 103, 85, 82, 94;
 * 7168 x 7168: 300 tokens 44.9, 45.9, 39.6, 46.4; 4096 tokens 301, 245, 254, 214.)
 */
struct TileCost {
    uint32_t bn, bt, alone, shared;
};
constexpr TileCost kTileCost[5] = {{128, 32, 420, 340}, {128, 64, 490, 390}, {128, 128, 750, 590},
                                   {256, 128, 1160, 1060}, {256, 256, 1900, 1800}};

Cut cut_of(uint32_t T, uint32_t N, uint32_t K) {
    const uint32_t groups = (K / kBlock + 3u) / 4u;
    Cut best{};
    const uint64_t room = parts_room(T, N, K);
    uint64_t least = ~0ull;
    for (int i = 0; i < 5; i++) {
        const TileCost &c = kTileCost[i];
        const uint32_t tt = (T + c.bt - 1u) / c.bt, tn = (N + c.bn - 1u) / c.bn;
        const uint64_t tiles = (uint64_t)tt * tn, padded = tiles * c.bt * c.bn;
        for (uint32_t want = 1u; want <= groups && want <= kMostSplits; want++) {
            if (want > 1u && (tiles * want > kMostCutBlocks || padded * want * 4u > room)) break;
            const uint32_t span = 4u * ((groups + want - 1u) / want);
            const uint32_t splits = (4u * groups + span - 1u) / span;
            if (splits != want) continue; /* the same cut as a smaller number's */
            const uint64_t each = (tiles * splits + 255u) / 256u;
            uint64_t ns = each * span * (each == 1u ? c.alone : c.shared);
            if (splits > 1u) ns += 3000u + padded * splits * 8u / 5000u;
            if (ns < least) {
                least = ns;
                best = Cut{i, tt, tn, splits, span};
            }
        }
    }
    return best;
}

template <class C>
bool launch_dense(TileArgs A, const Cut &q, hipStream_t st) {
    A.tiles_t = q.tiles_t, A.tiles_n = q.tiles_n, A.splits = q.splits, A.span = q.span;
    const uint32_t tiles = q.tiles_t * q.tiles_n;
    hipLaunchKernelGGL(product_tile_kernel<C>, dim3(8u * ((tiles * q.splits + 7u) / 8u)),
                       dim3(C::THREADS), 0, st, A);
    if (q.splits == 1u) return hipGetLastError() == hipSuccess;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(join_kernel<C>), dim3(tiles * 4u * C::TI), dim3(C::THREADS), 0,
                       st, A);
    return hipGetLastError() == hipSuccess;
}

/* The expert stage on given routes. */
bool run_fp8_experts(const Fp8Workspace &ws, void *output, const void *hidden, const void *residual,
                     const uint32_t *ids, const float *wts, const k3_moe_fp8_expert *experts,
                     const k3_moe_shape &s, uint32_t T, hipStream_t st) {
    const uint32_t H = s.hidden, F = s.ffn, E = s.expert_count, k = s.top_k;
    if (one_by_one(T, s)) {
        const OneExpertArgs A{experts, ids, wts, (const uint16_t *)hidden, (const uint16_t *)residual,
                              (uint16_t *)output, ws.h, H, F, E, k,
                              activation_of(s)};
        /* the waves' columns over the whole chip while they are few (8 experts of
         * 7168, 2048: 4 a block 41.8 us, 8 a block 48.9), 8 sharing a token's
         * codes where there are many (8 tokens of 2048, 512, 4 experts: 22 us, 1 a
         * block 27) */
        const uint32_t all = T * k * (F / 16u), waves = all <= 512u && H <= 2048u ? 1u : all <= 1024u ? 4u : 8u;
        const auto gateup = waves == 1u   ? gateup_one_kernel<1u, 16, 2048u>
                            : waves == 4u ? gateup_one_kernel<4u, 8, kOneHidden>
                                          : gateup_one_kernel<8u, 4, kOneHidden>;
        hipLaunchKernelGGL(gateup, dim3(T * k * (F / (16u * waves))), dim3(64u * waves), 0, st, A);
        if (F <= 2048u)
            hipLaunchKernelGGL(down_one_kernel<2048u>, dim3(H / 16u, T), dim3(512), 0, st, A);
        else
            hipLaunchKernelGGL(down_one_kernel<kOneFfn>, dim3(H / 16u, T), dim3(512), 0, st, A);
        return hipGetLastError() == hipSuccess;
    }
    const RowArgs R = row_args(ws.xq, ws.xs, hidden, T, H, scale_stride(H));
    const dim3 grid(1u + (uint32_t)((R.blocks + 63u) / 64u)); /* the plan's block, 64 blocks of rows each */
    if (T <= kSmallPlan) {
        const PlanArgs A{ws.lists, ws.token_index, ws.route_index, ids, experts, T, k, E, R};
        const bool few = (T + 63u) / 64u * E <= kFewWords;
        const auto plan = k <= 8u ? few ? small_plan_kernel<8, kFewWords> : small_plan_kernel<8, kMostWords>
                          : few   ? small_plan_kernel<32, kFewWords>
                                  : small_plan_kernel<32, kMostWords>;
        hipLaunchKernelGGL(plan, grid, dim3(1024), 0, st, A);
    } else {
        if (!k3_moe_route_plan(ws.counts, ws.offsets, ws.unique, ws.summary, ws.token_index,
                               ws.route_index, ids, T, k, E, ws.plan, ws.plan_bytes, st))
            return false;
        hipLaunchKernelGGL(tiles_kernel, grid, dim3(1024), 0, st, ws.lists, ws.counts, ws.offsets,
                           experts, E, R);
    }
    TileArgs B{};
    B.lists = ws.lists, B.token_index = ws.token_index, B.route_index = ws.route_index;
    B.xq = ws.xq, B.xs = ws.xs, B.xstride = scale_stride(H);
    B.out = ws.y, B.hq = ws.hq, B.hs = ws.hs, B.hstride = scale_stride(F);
    B.act = activation_of(s);
    B.N = F, B.K = H, B.tiles_n = F / kBlock;
    /* the classes' blocks are rounded up to eights */
    hipLaunchKernelGGL(experts_tile_kernel<kGateUp>, dim3(ws.tile_cap * B.tiles_n + 8u * kClasses),
                       dim3(512), 0, st, B);
    B.xq = ws.hq, B.xs = ws.hs, B.xstride = scale_stride(F);
    B.N = H, B.K = F, B.tiles_n = (H + 255u) / 256u;
    hipLaunchKernelGGL(experts_tile_kernel<kDown>, dim3(ws.tile_cap * B.tiles_n + 8u * kClasses),
                       dim3(512), 0, st, B);
    return hipGetLastError() == hipSuccess &&
           launch_combine(output, ws.y, residual, ids, wts, T, H, k, E, true, st);
}

/* 2^38 outputs (512 GiB) are half as many tiles as a launch takes: 2^23 blocks of 512
 * threads are 2^32. */
constexpr uint64_t kMostOutputs = 1ull << 38;
bool product_ok(uint32_t T, uint32_t rows, uint32_t cols) {
    return T != 0u && T <= 65535u && rows != 0u && rows <= kMostAxis && cols != 0u &&
           cols % kBlock == 0u && cols <= kMostAxis && (uint64_t)T * rows <= kMostOutputs;
}

size_t fp8_scratch_bytes(uint32_t T, uint32_t rows, uint32_t cols) {
    if (one_launch(T, rows, cols)) return 0u; /* encoded by the product's own kernel */
    return align256((size_t)T * cols) + align256(4u * (size_t)T * scale_stride(cols)) +
           parts_room(T, rows, cols);
}

}  // namespace

bool fp8_product_fits(uint32_t T, uint32_t rows, uint32_t cols) { return product_ok(T, rows, cols); }

}  // namespace k3

using namespace k3;

/* Blocks read their values and write codes and scales in no order. */
static bool encoded_apart(const uint8_t *codes, const float *scales, const void *src, uint64_t values,
                          uint64_t scale_count) {
    return !overlap(codes, values, src, 2u * values) && !overlap(scales, 4u * scale_count, src, 2u * values) &&
           !overlap(codes, values, scales, 4u * scale_count);
}

extern "C" bool k3_moe_fp8_128_quantize_rows_bf16(uint8_t *codes, float *scales, const void *src,
                                                  uint32_t rows, uint32_t columns, void *stream) {
    const uint64_t blocks = (uint64_t)rows * (columns / kBlock);
    if (!codes || !scales || !src || rows == 0u || columns == 0u || columns % kBlock != 0u ||
        blocks > (1ull << 34) || ((uintptr_t)src % 16u) != 0u || ((uintptr_t)codes % 8u) != 0u ||
        ((uintptr_t)scales % 4u) != 0u ||
        !encoded_apart(codes, scales, src, (uint64_t)rows * columns, blocks))
        return false;
    return launch_rows(row_args(codes, scales, src, rows, columns, columns / kBlock), (hipStream_t)stream);
}

extern "C" bool k3_moe_fp8_128_quantize_weight_bf16(uint8_t *codes, float *scales, const void *src,
                                                    uint32_t rows, uint32_t columns,
                                                    void *stream) {
    const uint64_t blocks = ((uint64_t)rows + kBlock - 1u) / kBlock * (columns / kBlock);
    if (!codes || !scales || !src || rows == 0u || columns == 0u || columns % kBlock != 0u ||
        blocks >= (1ull << 24) || /* 2^32 threads */
        ((uintptr_t)src % 16u) != 0u || ((uintptr_t)codes % 8u) != 0u ||
        ((uintptr_t)scales % 4u) != 0u ||
        !encoded_apart(codes, scales, src, (uint64_t)rows * columns, blocks))
        return false;
    hipLaunchKernelGGL(weight_kernel, dim3((uint32_t)blocks), dim3(256), 0, (hipStream_t)stream,
                       codes, scales, (const uint16_t *)src, rows, columns);
    return hipGetLastError() == hipSuccess;
}

extern "C" size_t k3_moe_fp8_128_scratch_bytes(uint32_t vector_count, uint32_t rows,
                                               uint32_t columns) {
    if (!product_ok(vector_count, rows, columns)) return 0u;
    return fp8_scratch_bytes(vector_count, rows, columns);
}

namespace {

/* The product of rows in bf16 (input), or encoded (xq, xs with a scale for each block). */
bool run_product(void *output, const uint8_t *codes, const float *scales, const void *input,
                 const uint8_t *xq, const float *xs, uint32_t T, uint32_t rows, uint32_t columns,
                 void *scratch, size_t scratch_bytes, hipStream_t st) {
    if (!output || !codes || !scales || !product_ok(T, rows, columns) ||
        (((uintptr_t)codes | (uintptr_t)input | (uintptr_t)xq) % 16u) != 0u ||
        (((uintptr_t)scales | (uintptr_t)xs) % 4u) != 0u || ((uintptr_t)output % 2u) != 0u)
        return false;
    /* blocks of one launch read all of the input and write their own columns */
    const uint64_t bytes = 2u * (uint64_t)T * rows, values = (uint64_t)T * columns;
    if (input ? overlap(output, bytes, input, 2u * values)
              : overlap(output, bytes, xq, values) || overlap(output, bytes, xs, values / kBlock * 4u))
        return false;
    const size_t need = fp8_scratch_bytes(T, rows, columns);
    if (need != 0u && (!scratch || scratch_bytes < need || ((uintptr_t)scratch % 256u) != 0u))
        return false;
    const bool wide = rows % 4u == 0u && ((uintptr_t)output % 8u) == 0u;
    if (one_launch(T, rows, columns)) {
        const OneArgs A{(uint16_t *)output, codes, scales, (const uint16_t *)input, xq, xs, T, rows,
                        columns};
        const auto pick = [&](auto encoded) {
            constexpr bool E = decltype(encoded)::value;
            return T == 1u   ? product_one_kernel<1u, 64u, E>
                   : T == 2u ? product_one_kernel<2u, 64u, E>
                   : T <= 4u ? product_one_kernel<4u, 64u, E>
                   : T <= 8u ? product_one_kernel<8u, 64u, E>
                             : product_one_kernel<16u, 32u, E>;
        };
        const auto product = input ? pick(std::false_type{}) : pick(std::true_type{});
        const dim3 grid((rows + 15u) / 16u, T <= 8u ? 1u : (T + 15u) / 16u);
        hipLaunchKernelGGL(product, grid, dim3(512), 0, st, A);
        return hipGetLastError() == hipSuccess;
    }
    TileArgs B{};
    uint8_t *const codes_at = (uint8_t *)scratch;
    float *const scales_at = (float *)(codes_at + align256((size_t)T * columns));
    B.codes = codes, B.scales = scales, B.xstride = scale_stride(columns);
    B.part = (f32x4 *)((uint8_t *)scales_at + align256(4u * (size_t)T * B.xstride));
    B.out = (uint16_t *)output, B.T = T, B.N = rows, B.K = columns, B.wide = wide;
    B.wide16 = rows % 8u == 0u && ((uintptr_t)output % 16u) == 0u;
    if (input) {
        B.xq = codes_at, B.xs = scales_at;
        if (!launch_rows(row_args(codes_at, scales_at, input, T, columns, B.xstride), st)) return false;
    } else {
        B.xq = xq, B.xs = xs;
        if (columns / kBlock != B.xstride || ((uintptr_t)xs % 16u) != 0u) { /* read four at a time */
            const uint64_t n = ((uint64_t)T * B.xstride + 255u) / 256u;
            hipLaunchKernelGGL(spread_scales_kernel, dim3((uint32_t)(n < 4096u ? n : 4096u)), dim3(256), 0,
                               st, scales_at, xs, T, columns / kBlock, B.xstride);
            if (hipGetLastError() != hipSuccess) return false;
            B.xs = scales_at;
        }
    }
    const Cut q = cut_of(T, rows, columns);
    switch (q.tile) {
    case 0: return launch_dense<Half32>(B, q, st);
    case 1: return launch_dense<Half64>(B, q, st);
    case 2: return launch_dense<Half128>(B, q, st);
    case 3: return launch_dense<Tile128>(B, q, st);
    default: return launch_dense<Tile256>(B, q, st);
    }
}

}  // namespace

extern "C" bool k3_moe_fp8_128_gemm_bf16(void *output, const uint8_t *codes, const float *scales,
                                         const void *input, uint32_t vector_count, uint32_t rows,
                                         uint32_t columns, void *scratch, size_t scratch_bytes,
                                         void *stream) {
    return input && run_product(output, codes, scales, input, nullptr, nullptr, vector_count, rows, columns,
                                scratch, scratch_bytes, (hipStream_t)stream);
}

extern "C" bool k3_moe_fp8_128_encoded_gemm_bf16(void *output, const uint8_t *codes,
                                                 const float *scales, const uint8_t *input_codes,
                                                 const float *input_scales, uint32_t vector_count,
                                                 uint32_t rows, uint32_t columns, void *scratch,
                                                 size_t scratch_bytes, void *stream) {
    return input_codes && input_scales &&
           run_product(output, codes, scales, nullptr, input_codes, input_scales, vector_count, rows, columns,
                       scratch, scratch_bytes, (hipStream_t)stream);
}

extern "C" size_t k3_moe_fp8_workspace_bytes(const k3_moe_shape *shape, uint32_t token_count) {
    return fp8_shape_ok(shape, token_count) ? carve(nullptr, *shape, token_count).bytes : 0u;
}

namespace {

bool fp8_args_ok(const void *output, const void *hidden, const void *residual,
                 const k3_moe_fp8_expert *experts, const k3_moe_shape *shape, uint32_t T,
                 const void *workspace) {
    if (!output || !hidden || !experts || !workspace || !fp8_shape_ok(shape, T)) return false;
    /* the last kernel's blocks read the residual and write the output, each its own
     * columns of a token; hidden has been read by then */
    const uint64_t bytes = 2u * (uint64_t)T * shape->hidden;
    if (residual && residual != output && overlap(output, bytes, residual, bytes)) return false;
    return (((uintptr_t)output | (uintptr_t)hidden | (uintptr_t)residual) % 16u) == 0u &&
           ((uintptr_t)experts % 8u) == 0u && ((uintptr_t)workspace % 256u) == 0u;
}

}  // namespace

extern "C" bool k3_moe_fp8_experts_bf16(void *output, const void *hidden, const void *residual,
                                        const void *expert_ids, const void *expert_weights,
                                        const k3_moe_fp8_expert *experts,
                                        const k3_moe_shape *shape, uint32_t token_count,
                                        void *workspace, size_t workspace_bytes, void *stream) {
    if (!expert_ids || !expert_weights ||
        (((uintptr_t)expert_ids | (uintptr_t)expert_weights) % 4u) != 0u ||
        !fp8_args_ok(output, hidden, residual, experts, shape, token_count, workspace))
        return false;
    const Fp8Workspace ws = carve(workspace, *shape, token_count);
    if (workspace_bytes < ws.bytes) return false;
    return run_fp8_experts(ws, output, hidden, residual, (const uint32_t *)expert_ids,
                           (const float *)expert_weights, experts, *shape, token_count,
                           (hipStream_t)stream);
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
    return run_fp8_experts(ws, output, hidden, residual, ws.ids, ws.weights, experts, s, token_count,
                           st);
}
