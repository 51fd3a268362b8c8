/*
 * The router in training: balance loss with per-expert counts, and the gradient
 * by the router's logits (include/k3_moe.h has the formulas; the reference only
 * serves and has no counterpart).
 *
 *   balance_part_kernel    a block: a run of one segment's tokens, a token a
 *                          wave at a time; sums of the shares sigma / Z and
 *                          the counts of its run
 *   balance_join_kernel    joins the runs, writes counts and mean scores; the
 *                          last block to end adds up the loss
 *   balance_loss_kernel    adds up the loss of segments of one run each
 *   router_backward_kernel a token a wave at a time, the segment's f in
 *                          registers
 *
 * Expert e of a row is slot e / 64 of lane e % 64. All sums run in an order set
 * by the sizes: counts are whole numbers, and the last block reads every
 * partial loss in one order whichever block it is.
 */
#include "k3_device.h"
#include "k3_internal.h"
#include "../../include/k3_moe.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace k3 {
namespace {

constexpr uint32_t kWaves = 8;  /* of a block of balance_part_kernel */
constexpr uint32_t kJoin = 16;  /* experts of a block of balance_join_kernel */
constexpr uint32_t kBackWaves = 4;

inline size_t align256(size_t v) { return (v + 255u) & ~(size_t)255u; }

/* sigma(x) = 1 / (1 + t), t = e^-x, to (8 + 2 |x|) 2^-24 of itself: the exponent is one
 * rounded product, off by |x| 2^-24 of t, the rest a few ulp. 0 where it would be under
 * 2^-126 (x < -87.33), which the hardware's reciprocal gives as 0. */
__device__ __forceinline__ float exp_neg(float x) {
    return __builtin_amdgcn_exp2f(__fmul_rn(x, -1.44269504088896341f));
}
__device__ __forceinline__ float sigma_of(float t) {
    return __builtin_amdgcn_rcpf(__fadd_rn(1.0f, t));
}
/* sigma (1 - sigma) = t sigma^2: no difference of near values, and 0 where sigma
 * is 0. */
__device__ __forceinline__ float slope_of(float t, float sigma) {
    return __fmul_rn(__fmul_rn(fminf(t, 0x1p126f), sigma), sigma);
}

/* Lane r < k: the id of route r of a token; E past them. */
__device__ __forceinline__ uint32_t load_ids(const uint32_t *ids, uint64_t t, uint32_t k, uint32_t E) {
    const uint32_t lane = threadIdx.x & 63u;
    return lane < k ? ids[t * k + lane] : E;
}
/* The route of lane r < k of a token by load_ids: its id, or E where it has none
 * (no such rank, an id from E on, or one that an earlier rank has). */
__device__ __forceinline__ uint32_t lane_route(uint32_t id, uint32_t k, uint32_t E) {
    const uint32_t lane = threadIdx.x & 63u;
    bool again = id >= E;
    for (uint32_t r = 0; r + 1u < k; r++)
        again |= lane > r && id == (uint32_t)__builtin_amdgcn_readlane((int)id, (int)r);
    return again ? E : id;
}

/* Slots of a row of J that are whole wherever with_slots picks J. */
constexpr int whole_slots(int J) { return J <= 4 ? J - 1 : J - 2; }

/* The logits of token t (-inf, score 0, past E). */
template <int J>
__device__ __forceinline__ void load_row(float (&x)[J], const float *logits, uint64_t t,
                                         uint32_t E) {
    const uint32_t lane = threadIdx.x & 63u;
    const float *row = logits + t * E;
#pragma unroll
    for (int j = 0; j < J; j++) {
        const uint32_t e = lane + 64u * (uint32_t)j;
        x[j] = j < whole_slots(J) || e < E ? row[e] : -__builtin_huge_valf();
    }
}

struct BalanceArgs {
    float *loss;
    uint32_t *counts;
    float *mean;
    uint32_t *live;
    const float *logits;
    const uint32_t *ids;
    const uint8_t *mask;
    uint32_t S, L, E, k;
    float coef;
    uint32_t runs, span; /* runs of `span` tokens of a segment */
    float *part_mean;    /* [S, runs, E] */
    uint32_t *part_count;
    uint32_t *part_live; /* [S, runs] */
    float *part_loss;    /* [S, ceil(E / kJoin)] */
    uint32_t *ticket;
};

/* Expert e of segment s, with the sum m of its shares and its count c: written, and
 * its term of the loss. n: the segment's live tokens. */
__device__ __forceinline__ float close_expert(const BalanceArgs &A, uint32_t s, uint32_t e, float m,
                                              uint32_t c, uint32_t n) {
    m = n ? __fdiv_rn(m, (float)n) : 0.0f;
    A.counts[(uint64_t)s * A.E + e] = c;
    A.mean[(uint64_t)s * A.E + e] = m;
    return n ? __fmul_rn(__fdiv_rn(__fmul_rn((float)c, (float)A.E), __fmul_rn((float)A.k, (float)n)), m)
             : 0.0f;
}
/* The sum of v over a block of WAVES waves, in thread 0. */
template <uint32_t WAVES>
__device__ __forceinline__ float block_sum(float v) {
    __shared__ float part[WAVES];
    v = wave_sum(v);
    if ((threadIdx.x & 63u) == 0u) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < WAVES; w++) v = __fadd_rn(v, part[w]);
    return v;
}
/* The loss from `n` partial ones, by a block of 1024 threads. */
__device__ __forceinline__ void close_loss(const BalanceArgs &A, uint32_t n) {
    float v = 0.0f;
    for (uint32_t q = threadIdx.x; q < n; q += 1024u)
        v = __fadd_rn(v, __hip_atomic_load(&A.part_loss[q], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    v = block_sum<16>(v);
    if (threadIdx.x == 0u) *A.loss = __fmul_rn(v, __fdiv_rn(A.coef, (float)A.S));
}

/* WHOLE: a run is a segment, and the block writes what is the segment's. A row is
 * read once into registers, where the wave adds up its scores and scales them.
 * 8192 tokens of 896 experts: 11.5 us, 2.6 TB/s; of 64 experts the wave's sums over
 * its lanes bound it (262144 tokens 54 us). */
template <int J, bool WHOLE>
__global__ __launch_bounds__(64 * kWaves) void balance_part_kernel(BalanceArgs A) {
    __shared__ float sums[kWaves][64 * J];
    __shared__ uint32_t hist[64 * J];
    __shared__ uint32_t lives[kWaves];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, E = A.E;
    const uint32_t s = blockIdx.x / A.runs, run = blockIdx.x % A.runs;
    const uint32_t i0 = run * A.span, i1 = min(i0 + A.span, A.L);
    if (!WHOLE && blockIdx.x == 0u && threadIdx.x == 0u) *A.ticket = 0u; /* for the next kernel */
    for (uint32_t e = threadIdx.x; e < 64u * J; e += 64u * kWaves) hist[e] = 0u;
    __syncthreads();
    float acc[J];
#pragma unroll
    for (int j = 0; j < J; j++) acc[j] = 0.0f;
    uint32_t live = 0u;
    for (uint32_t i = i0 + wave; i < i1; i += kWaves) {
        const uint64_t t = (uint64_t)s * A.L + i;
        if (A.mask && A.mask[t] == 0u) continue;
        live++;
        float x[J];
        const uint32_t id = load_ids(A.ids, t, A.k, E);
        load_row<J>(x, A.logits, t, E);
        const uint32_t e = lane_route(id, A.k, E);
        if (e < E) atomicAdd(&hist[e], 1u);
        float z = 0.0f;
#pragma unroll
        for (int j = 0; j < J; j++) {
            x[j] = sigma_of(exp_neg(x[j]));
            z = __fadd_rn(z, x[j]);
        }
        z = wave_sum(z);
        const float inv = z == 0.0f ? 0.0f : __fdiv_rn(1.0f, z);
#pragma unroll
        for (int j = 0; j < J; j++) acc[j] = fmaf(x[j], inv, acc[j]);
    }
#pragma unroll
    for (int j = 0; j < J; j++) sums[wave][64 * j + lane] = acc[j];
    if (lane == 0u) lives[wave] = live;
    __syncthreads();
    uint32_t n = 0u;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; w++) n += lives[w];
    const uint64_t at = (uint64_t)blockIdx.x * E;
    float l = 0.0f;
    for (uint32_t e = threadIdx.x; e < E; e += 64u * kWaves) {
        float v = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kWaves; w++) v = __fadd_rn(v, sums[w][e]);
        if constexpr (WHOLE) {
            l = __fadd_rn(l, close_expert(A, s, e, v, hist[e], n));
        } else {
            A.part_mean[at + e] = v;
            A.part_count[at + e] = hist[e];
        }
    }
    if constexpr (WHOLE) l = block_sum<kWaves>(l);
    if (threadIdx.x != 0u) return;
    if constexpr (WHOLE) {
        A.live[s] = n;
        if (A.S == 1u)
            *A.loss = __fmul_rn(l, A.coef);
        else
            A.part_loss[s] = l;
    } else {
        A.part_live[blockIdx.x] = n;
    }
}

/* The loss of segments whose blocks were whole: thousands of tickets would cost
 * more than this launch (4096 segments of 64 tokens: 353 us with tickets). */
__global__ __launch_bounds__(1024) void balance_loss_kernel(BalanceArgs A) { close_loss(A, A.S); }

/* Joins the runs of a segment: 16 experts a block, 64 runs at a time, or (WIDE) all
 * experts of a segment a block; the last block to end closes the loss. 5.8 us for
 * 512 runs of 896 experts: the latency of a read, of the ticket and of the partial
 * losses. */
template <bool WIDE>
__global__ __launch_bounds__(1024) void balance_join_kernel(BalanceArgs A) {
    __shared__ float fsum[16][kJoin];
    __shared__ uint32_t csum[16][kJoin];
    __shared__ uint32_t nsum[16];
    __shared__ uint32_t last;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, E = A.E;
    float m = 0.0f, l = 0.0f;
    uint32_t c = 0u, n = 0u;
    if constexpr (WIDE) {
        const uint32_t s = blockIdx.x, e = threadIdx.x;
        const uint64_t at = (uint64_t)s * A.runs * E + e;
        for (uint32_t r = 0; r < A.runs; r++) n += A.part_live[s * A.runs + r];
        if (e < E) {
#pragma unroll 8
            for (uint32_t r = 0; r < A.runs; r++) {
                m = __fadd_rn(m, A.part_mean[at + (uint64_t)r * E]);
                c += A.part_count[at + (uint64_t)r * E];
            }
            l = close_expert(A, s, e, m, c, n);
        }
        if (e == 0u) A.live[s] = n;
        l = block_sum<16>(l);
    } else {
        const uint32_t cols = (E + kJoin - 1u) / kJoin, s = blockIdx.x / cols;
        const uint32_t i = lane % kJoin, e = kJoin * (blockIdx.x % cols) + i;
        for (uint32_t r = threadIdx.x; r < A.runs; r += 1024u) n += A.part_live[s * A.runs + r];
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) n += __shfl_xor(n, o, 64);
        if (e < E) {
            const uint64_t at = (uint64_t)s * A.runs * E + e;
#pragma unroll 8
            for (uint32_t r = threadIdx.x / kJoin; r < A.runs; r += 1024u / kJoin) {
                m = __fadd_rn(m, A.part_mean[at + (uint64_t)r * E]);
                c += A.part_count[at + (uint64_t)r * E];
            }
        }
#pragma unroll
        for (int o = kJoin; o < 64; o <<= 1) {
            m = __fadd_rn(m, __shfl_xor(m, o, 64));
            c += __shfl_xor(c, o, 64);
        }
        if (lane < kJoin) fsum[wave][i] = m, csum[wave][i] = c;
        if (lane == 0u) nsum[wave] = n;
        __syncthreads();
        if (wave == 0u) {
            m = 0.0f, c = 0u, n = 0u;
#pragma unroll
            for (uint32_t w = 0; w < 16u; w++) {
                m = __fadd_rn(m, fsum[w][i]);
                c += csum[w][i];
                n += nsum[w];
            }
            if (e < E && lane < kJoin) l = close_expert(A, s, e, m, c, n);
            if (e == 0u && lane == 0u) A.live[s] = n;
            l = wave_sum(l);
        }
    }
    if (threadIdx.x == 0u) {
        __hip_atomic_store(&A.part_loss[blockIdx.x], l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = __hip_atomic_fetch_add(A.ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) ==
               gridDim.x - 1u;
    }
    __syncthreads();
    if (last) close_loss(A, gridDim.x);
}

struct BackwardArgs {
    float *out;
    const float *logits;
    const uint32_t *ids, *counts, *live;
    const uint8_t *mask;
    const float *dloss, *dw;
    uint32_t S, L, E, k;
    float coef, scale;
    uint32_t runs, span;
};

/* A row in registers again, its two sums, its gradient. Its lanes store every expert
 * that the token did not choose, and lane r the one of route r, whose score it
 * reads again (from the cache): handed over through LDS, rows of 64 KB a block
 * left two blocks a CU and took 27 us for 8192 tokens of 896 experts, 19.2 here (3.1
 * TB/s read and written; four waves' sums over their lanes hide the loads). */
template <int J>
__global__ __launch_bounds__(64 * kBackWaves) void router_backward_kernel(BackwardArgs A) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, E = A.E;
    const uint32_t s = blockIdx.x / A.runs, run = blockIdx.x % A.runs;
    const uint32_t i0 = run * A.span, i1 = min(i0 + A.span, A.L);
    const uint32_t n = A.live[s];
    const uint32_t *counts = A.counts + (uint64_t)s * E;
    /* f, and the factor that the loss has in common: both 0 without live tokens. The
     * factor does not meet 1 / Z before the slope has: scores near 2^-126 and a large
     * loss_gradient would take that past fp32, while slope / Z <= 1. */
    const float per = n ? __fdiv_rn((float)E, __fmul_rn((float)A.k, (float)n)) : 0.0f;
    float share = n ? __fdiv_rn(__fdiv_rn(A.coef, (float)A.S), (float)n) : 0.0f;
    if (A.dloss) share = __fmul_rn(share, *A.dloss);
    float f[J];
#pragma unroll
    for (int j = 0; j < J; j++) {
        const uint32_t e = lane + 64u * (uint32_t)j;
        f[j] = e < E ? __fmul_rn((float)counts[e], per) : 0.0f;
    }
    for (uint32_t i = i0 + wave; i < i1; i += kBackWaves) {
        const uint64_t t = (uint64_t)s * A.L + i;
        float *out = A.out + t * E;
        if (A.mask && A.mask[t] == 0u) {
#pragma unroll
            for (int j = 0; j < J; j++)
                if (lane + 64u * (uint32_t)j < E) out[lane + 64u * (uint32_t)j] = 0.0f;
            continue;
        }
        float x[J], d[J];
        /* the ids first: the loads that go by them wait for nothing else */
        const uint32_t id = A.dw ? load_ids(A.ids, t, A.k, E) : E;
        asm volatile("" ::: "memory");
        load_row<J>(x, A.logits, t, E);
        /* lane r: route r's expert (E: none), its logit, f and gradient */
        uint32_t e = E;
        float xe = -__builtin_huge_valf(), fe = 0.0f, dw = 0.0f;
        if (A.dw) {
            e = lane_route(id, A.k, E);
            if (e < E) {
                xe = A.logits[t * E + e];
                fe = __fmul_rn((float)counts[e], per);
                dw = A.dw[t * A.k + lane];
            }
        }
        float z = 0.0f, a = 0.0f;
#pragma unroll
        for (int j = 0; j < J; j++) {
            const float u = exp_neg(x[j]), p = sigma_of(u);
            d[j] = slope_of(u, p);
            z = __fadd_rn(z, p);
            a = fmaf(f[j], p, a);
        }
        z = wave_sum(z);
        a = wave_sum(a);
        const float inv = z == 0.0f ? 0.0f : __fdiv_rn(1.0f, z);
        const float mean = __fmul_rn(a, inv);
        uint32_t chosen = 0u; /* the slots of this lane that a route has */
        if (A.dw) {
            for (uint32_t r = 0; r < A.k; r++) {
                const uint32_t er = (uint32_t)__builtin_amdgcn_readlane((int)e, (int)r);
                chosen |= er < E && (er & 63u) == lane ? 1u << (er >> 6) : 0u;
            }
            const float u = exp_neg(xe), p = sigma_of(u); /* 0 without a route */
            const float den = __fadd_rn(wave_sum(p), 1e-20f);
            const float m = __fdiv_rn(wave_sum(__fmul_rn(dw, p)), den);
            const float add = __fmul_rn(__fdiv_rn(A.scale, den), __fsub_rn(dw, m));
            const float d = slope_of(u, p);
            if (e < E)
                out[e] = __fadd_rn(__fmul_rn(__fmul_rn(share, __fsub_rn(fe, mean)), __fmul_rn(d, inv)),
                                   __fmul_rn(add, d));
        }
#pragma unroll
        for (int j = 0; j < J; j++) {
            const uint32_t q = lane + 64u * (uint32_t)j;
            if ((j < whole_slots(J) || q < E) && !(chosen >> j & 1u))
                out[q] = __fmul_rn(__fmul_rn(share, __fsub_rn(f[j], mean)), __fmul_rn(d[j], inv));
        }
    }
}

/* Two blocks a CU read a batch (their partial sums are another eighth of the
 * reads at 8192 tokens), four write its gradient. */
constexpr uint32_t kPartBlocks = 512, kBackBlocks = 1024;
/* Joins of a whole segment a block: of up to 16 runs, and where 16 experts a block
 * would be more blocks than the chip holds at once (30 segments of 300 tokens,
 * 1024 experts: loss 54 us so, 18.5 here). */
constexpr uint32_t kFewRuns = 16, kJoinBlocks = 512;

/* Runs a segment is cut into: about `blocks` in all, of `waves` tokens at
 * least. */
uint32_t most_runs(uint32_t S, uint32_t L, uint32_t blocks, uint32_t waves) {
    const uint32_t want = (blocks + S - 1u) / S, most = (L + waves - 1u) / waves;
    return want < most ? want : most;
}
void runs_of(uint32_t S, uint32_t L, uint32_t blocks, uint32_t waves, uint32_t &runs, uint32_t &span) {
    runs = most_runs(S, L, blocks, waves);
    span = (L + runs - 1u) / runs;
    runs = (L + span - 1u) / span;
}

bool batch_ok(uint32_t S, uint32_t L, uint32_t E) {
    return S != 0u && S <= 65535u && L != 0u && (uint64_t)S * L <= (1ull << 24) && E != 0u &&
           E <= 1024u;
}

size_t carve(BalanceArgs &A, void *base) {
    uint8_t *p = (uint8_t *)base;
    size_t off = 0;
    auto take = [&](size_t n) {
        uint8_t *q = p ? p + off : nullptr;
        off += align256(n);
        return q;
    };
    /* grows with the length: scratch of longer segments serves shorter ones */
    const size_t parts = (size_t)A.S * most_runs(A.S, A.L, kPartBlocks, kWaves);
    A.part_mean = (float *)take(4u * parts * A.E);
    A.part_count = (uint32_t *)take(4u * parts * A.E);
    A.part_live = (uint32_t *)take(4u * parts);
    A.part_loss = (float *)take(4u * (size_t)A.S * ((A.E + kJoin - 1u) / kJoin));
    A.ticket = (uint32_t *)take(4u);
    return off;
}

/* f(integral_constant<int, J>) for the least J here with E <= 64 J */
template <int J = 1, class F>
void with_slots(uint32_t E, F &&f) {
    constexpr int next = J < 4 ? J + 1 : J + 2;
    if constexpr (J < 16) {
        if (E > 64u * J) return with_slots<next>(E, f);
    }
    f(std::integral_constant<int, J>{});
}

}  // namespace
}  // namespace k3

using namespace k3;

extern "C" size_t k3_moe_balance_scratch_bytes(uint32_t segments, uint32_t length,
                                               uint32_t expert_count) {
    if (!batch_ok(segments, length, expert_count)) return 0u;
    BalanceArgs A{};
    A.S = segments, A.L = length, A.E = expert_count;
    runs_of(segments, length, kPartBlocks, kWaves, A.runs, A.span);
    return carve(A, nullptr);
}

extern "C" bool k3_moe_balance_loss_f32(float *loss, uint32_t *counts, float *mean_scores,
                                        uint32_t *live_tokens, const float *logits,
                                        const uint32_t *expert_ids, const uint8_t *mask,
                                        uint32_t segments, uint32_t length, uint32_t expert_count,
                                        uint32_t top_k, float coefficient, void *scratch,
                                        size_t scratch_bytes, void *stream) {
    if (!loss || !counts || !mean_scores || !live_tokens || !logits || !expert_ids || !scratch ||
        !batch_ok(segments, length, expert_count) || top_k == 0u || top_k > 32u ||
        top_k > expert_count || ((uintptr_t)scratch % 256u) != 0u ||
        scratch_bytes < k3_moe_balance_scratch_bytes(segments, length, expert_count))
        return false;
    BalanceArgs A{loss, counts, mean_scores, live_tokens, logits, expert_ids, mask, segments, length,
                  expert_count, top_k, coefficient};
    runs_of(segments, length, kPartBlocks, kWaves, A.runs, A.span);
    carve(A, scratch);
    const hipStream_t st = (hipStream_t)stream;
    with_slots(expert_count, [&](auto J) {
        constexpr int j = decltype(J)::value;
        const auto part = A.runs == 1u ? balance_part_kernel<j, true> : balance_part_kernel<j, false>;
        hipLaunchKernelGGL(part, dim3(segments * A.runs), dim3(64u * kWaves), 0, st, A);
    });
    const uint32_t blocks = segments * ((expert_count + kJoin - 1u) / kJoin); /* of 16 experts */
    if (A.runs == 1u) {
        if (segments > 1u) hipLaunchKernelGGL(balance_loss_kernel, dim3(1), dim3(1024), 0, st, A);
    } else if (A.runs <= kFewRuns || blocks > kJoinBlocks) {
        hipLaunchKernelGGL(balance_join_kernel<true>, dim3(segments), dim3(1024), 0, st, A);
    } else {
        hipLaunchKernelGGL(balance_join_kernel<false>, dim3(blocks), dim3(1024), 0, st, A);
    }
    return hipGetLastError() == hipSuccess;
}

extern "C" bool k3_moe_router_backward_f32(float *logits_gradient, const float *logits,
                                           const uint32_t *expert_ids, const uint32_t *counts,
                                           const uint32_t *live_tokens, const uint8_t *mask,
                                           const float *loss_gradient,
                                           const float *weight_gradient, uint32_t segments,
                                           uint32_t length, uint32_t expert_count, uint32_t top_k,
                                           float coefficient, float scaling_factor, void *stream) {
    if (!logits_gradient || !logits || !counts || !live_tokens ||
        (weight_gradient && !expert_ids) || !batch_ok(segments, length, expert_count) ||
        top_k == 0u || top_k > 32u || top_k > expert_count || !(scaling_factor > 0.0f))
        return false;
    /* a wave reads its row whole before it writes it, and no other row */
    const uint64_t bytes = 4ull * segments * length * expert_count;
    if (logits_gradient != logits && overlap(logits_gradient, bytes, logits, bytes)) return false;
    BackwardArgs A{logits_gradient, logits, expert_ids, counts, live_tokens, mask, loss_gradient,
                   weight_gradient, segments, length, expert_count, top_k, coefficient,
                   scaling_factor, 0u, 0u};
    runs_of(segments, length, kBackBlocks, kBackWaves, A.runs, A.span);
    with_slots(expert_count, [&](auto J) {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(router_backward_kernel<decltype(J)::value>),
                           dim3(segments * A.runs), dim3(64u * kBackWaves), 0, (hipStream_t)stream, A);
    });
    return hipGetLastError() == hipSuccess;
}
