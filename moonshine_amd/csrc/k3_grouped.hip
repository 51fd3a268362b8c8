/*
 * bf16 products grouped by expert: rows offsets[e] .. offsets[e + 1] belong to
 * expert e, as k3_moe_route_plan sorts them. No reference counterpart (the
 * reference only serves, on MXFP4 experts); the formulas are in
 * include/k3_moe.h.
 *
 *   product          y[r, n]     = sum_k x[r, k] W[e, n, k]
 *   input gradient   dx[r, k]    = sum_n dy[r, n] W[e, n, k]
 *   weight gradient  dW[e, n, k] = sum_r dy[r, n] x[r, k]
 *
 * All three are D[p, q] = sum over a reduction z of P[p, z] Q[q, z], P the
 * first operand of V_MFMA_F32_16X16X32_BF16 and Q the second, so that a lane of
 * the result holds four consecutive p, which lie side by side in the output:
 *
 *                    p   q   z    P in memory        Q in memory
 *   product          n   r   k    rows (z inside)    rows
 *   input gradient   k   r   n    columns (p inside) rows
 *   weight gradient  k   n   r    columns            columns
 *
 * An operand of rows is staged in LDS as its 128-byte pieces (64 z) and read 16
 * bytes a lane; one of columns as 64 rows of z (the weight gradient: 32), and read by the transposing LDS
 * load (ds_read_b64_tr_b16: of 16 lanes that address four rows of 16 values,
 * lane c gets column c). Products are exact in fp32 and summed in fp32.
 */
#include "k3_device.h"
#include "k3_internal.h"
#include "k3_lds.h"
#include "../../include/k3_moe.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace k3 {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));

/* Widths, and rows that an index picks from, are addressed by 32 bits. */
constexpr uint32_t kMostWidth = 1u << 15, kMostPicked = 65535, kMostRows = 65535u * 32u;
constexpr uint32_t kDepth = 64; /* z of a stage */

enum Direction { kProduct, kInput };

struct GroupArgs {
    const uint16_t *p, *q;     /* the operands: W and rows; weight gradient: x and dy */
    const uint32_t *offsets;   /* [E + 1] */
    const uint32_t *p_index, *q_index; /* rows of p (weight gradient), q; NULL: as they lie */
    const uint32_t *to;        /* output rows; NULL: as they lie */
    uint32_t p_rows, q_rows, to_rows; /* indices below these are rows */
    void *out;
    uint32_t R, E;
    uint32_t P, Z, Q;          /* p; z (weight gradient: unused); weight gradient: q */
    uint32_t tiles_p, tiles_q;
    bool accumulate;
};

/*
 * Memory for loads to LDS by 32-bit offsets: a lane's address is one register (of 64-bit
 * addresses their arithmetic took a fifth of a stage), and what lies at `bytes` or beyond
 * reads as zeros, as the ends of a reduction have to.
 */
constexpr uint32_t kNowhere = 0xfffffff0u;
struct Range {
    const uint8_t *base;
    uint32_t bytes;
    __device__ __forceinline__ Range() {}
    __device__ __forceinline__ Range(const void *p, uint64_t size)
        : base((const uint8_t *)p), bytes((uint32_t)(size < kNowhere ? size : kNowhere)) {}
    template <int Bytes>
    __device__ __forceinline__ void load(uint32_t at, uint8_t *lds) const {
        const __amdgpu_buffer_rsrc_t r =
            __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, (int)bytes, 0x00027000);
        if constexpr (Bytes == 16)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void *)lds, 16, (int)at, 0, 0, 0);
        else
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void *)lds, 4, (int)at, 0, 0, 0);
    }
};

__device__ __forceinline__ uint2 bf16x4(const f32x4 &v) {
    return make_uint2(bf16_pack2(v[0], v[1]), bf16_pack2(v[2], v[3]));
}

/* Rows of each but the last of an expert's tiles: all of up to 128 rows in one, more
 * in as few tiles of at most 256 as hold them, of whole steps of 32 rows. */
__device__ __forceinline__ uint32_t tile_height(uint32_t n) {
    const uint32_t steps = (n + 31u) / 32u, many = (n + 255u) / 256u;
    return n > 128u ? 32u * ((steps + many - 1u) / many) : n;
}

/* Expert e's rows [begin, begin + n) by the offsets; offsets that do not ascend,
 * or pass R, are cut so that no row lies outside. */
__device__ __forceinline__ uint32_t rows_of(const uint32_t *offsets, uint32_t e, uint32_t R,
                                            uint32_t &begin) {
    const uint32_t end = min(offsets[e + 1u], R);
    begin = min(offsets[e], R);
    return end > begin ? end - begin : 0u;
}

/* Sums over the lanes up to each. */
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, false); /* row_shr 1, 2, 4, 8 */
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false); /* row_bcast 15, 31 */
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);
    return v;
}

struct RowTile {
    uint32_t expert, row, rows, n; /* n: all rows of the expert */
};

/*
 * Row tile and column of work `block` among all experts' row tiles (of MOST rows at most) x
 * tiles_p columns, found by every wave for itself from the offsets: each lane counts the
 * tiles of up to 16 consecutive experts, and the lanes then take those of the one that holds
 * the tile. About 1 us at 64 experts, where a launch that lists the tiles takes 4; past
 * that a lane's experts are a load after the other: a launch that only looks its 256 tiles up takes 4.0 us
 * of 64 experts, 3.7 of 128, 5.9 of 256, 13.5 of 512 and 31.5 of 896, and the products of 32 rows each of 64
 * of them, 1024 x 512, 14.0 us of 64 and 42.7 of 896. Where most experts have rows it is less of the whole:
 * 1024 rows of 613 of 896 experts of 1024 x 1024 230 us, of which their weights take 211. An expert's tiles
 * of one column are neighbours, as they read the same weights; XCD x (blocks x,
 * x + 8, ...) takes a contiguous range of the works. False past the end.
 */
template <uint32_t MOST>
__device__ __forceinline__ bool find_tile(const GroupArgs &A, uint32_t block, RowTile &t,
                                          uint32_t &col) {
    const uint32_t lane = threadIdx.x & 63u, per = (A.E + 63u) / 64u;
    uint32_t mine = 0u, begin = 0u, n = 0u;
    for (uint32_t i = 0; i < per; i++) {
        const uint32_t e = lane * per + i;
        n = e < A.E ? rows_of(A.offsets, e, A.R, begin) : 0u;
        mine += (n + MOST - 1u) / MOST;
    }
    const uint32_t upto = wave_scan(mine);
    const uint32_t works = __builtin_amdgcn_readlane(upto, 63) * A.tiles_p, each = (works + 7u) / 8u;
    const uint32_t w = (block & 7u) * each + (block >> 3);
    if ((block >> 3) >= each || w >= works) return false;
    const uint32_t tile = w / A.tiles_p; /* an expert's tiles x columns, before its order is set */
    const uint32_t owner = __builtin_ctzll(__ballot(upto > tile));
    uint32_t at = owner, first = __builtin_amdgcn_readlane(upto - mine, owner), many = mine;
    if (per > 1u) {
        const uint32_t e = owner * per + lane;
        n = lane < per && e < A.E ? rows_of(A.offsets, e, A.R, begin) : 0u;
        many = (n + MOST - 1u) / MOST;
        const uint32_t to = first + wave_scan(many);
        at = __builtin_ctzll(__ballot(to > tile));
        first = __builtin_amdgcn_readlane(to - many, at);
    }
    t.n = __builtin_amdgcn_readlane(n, at);
    many = __builtin_amdgcn_readlane(many, at);
    t.expert = per > 1u ? owner * per + at : at;
    const uint32_t local = (tile - first) * A.tiles_p + w % A.tiles_p;
    const uint32_t height = MOST == 256u ? tile_height(t.n) : MOST, index = local % many;
    col = local / many;
    t.row = __builtin_amdgcn_readlane(begin, at) + height * index;
    t.rows = min(height, t.n - height * index);
    return true;
}

/* 64 WN of p x 32 TI of q a block of 2 WN waves; wave (wn, wt) holds p 64 wn .. + 64
 * and the subtiles (16 q) wt, wt + 2, ... */
template <int DIR_, int WN_, int TI_, int STAGES_>
struct Tile {
    static constexpr int DIR = DIR_, WN = WN_, TI = TI_, STAGES = STAGES_, WAVES = 2 * WN,
                         THREADS = 64 * WAVES;
    static constexpr bool PCOLS = DIR != kProduct;
    static constexpr uint32_t BP = 64 * WN, BQ = 32 * TI;
    static constexpr uint32_t A = BP * kDepth * 2, B = BQ * kDepth * 2, STAGE = A + B;
    static constexpr uint32_t B_CHUNKS = 4 * TI; /* of 1 KB; fewer than the waves: some load the same */
    static constexpr int DA = 4, DB = B_CHUNKS < WAVES ? 1 : B_CHUNKS / WAVES, D = DA + DB;
    static constexpr uint32_t LDS = STAGES * STAGE;
    static_assert(LDS <= 160u * 1024u, "LDS");
    /* Two stages: P, and the first 128 q (four subtiles of a wave, which take half of Q's
     * loads), are in registers or done with before the fourth subtile's products, so behind
     * a second barrier there their places take those of two stages on; the other q's follow
     * in the next stage. */
    static constexpr bool EARLY = STAGES == 2;
    static constexpr int HALF = EARLY ? DB / 2 : 0; /* loads of the first panel */
    static_assert(!EARLY || (TI == 8 && HALF * WAVES == 16), "two panels of 128 q");
    static __device__ __forceinline__ uint32_t b_chunk(uint32_t wave, uint32_t q) {
        if constexpr (EARLY) return 16u * (q / HALF) + HALF * wave + q % HALF;
        return B_CHUNKS < WAVES ? wave % B_CHUNKS : DB * wave + q;
    }
};

/*
 * Columns: row z of a stage is 2 B bytes (B the operand's width), a subtile of 16
 * columns 32 of them, a unit. Unit u of row z lies at unit u ^ s(z), so that the eight
 * rows 8 g + j (j < 4, g of one parity or the other) that 32 lanes read at once
 * lie in different banks (64 of 4 bytes: eight units).
 */
template <uint32_t B>
__device__ __forceinline__ uint32_t col_swizzle(uint32_t z) {
    static_assert(B >= 128u, "eight units a row");
    return (z & 3u) | (z >> 3 & 1u) << 2;
}
/* Chunk ch (1 KB) of a stage: lane L's z, and its source's 16-byte piece of that row. */
template <uint32_t B>
__device__ __forceinline__ uint32_t col_dma_z(uint32_t L, uint32_t ch) { return ch * (512u / B) + L / (B / 8u); }
template <uint32_t B>
__device__ __forceinline__ uint32_t col_dma_piece(uint32_t L, uint32_t ch) {
    const uint32_t piece = L % (B / 8u), s = col_swizzle<B>(col_dma_z<B>(L, ch));
    return (piece >> 1 ^ s) << 1 | (piece & 1u);
}
/* A lane's place for the reads of unit 0: z = 8 g + j, its 8 bytes of four columns.
 * Unit u's is this ^ 32 u; z + 4 and z + 32 lie 8 B and 64 B bytes on. */
template <uint32_t B>
__device__ __forceinline__ uint32_t col_slot(uint32_t lane) {
    const uint32_t z = 8u * (lane >> 4) + (lane >> 2 & 3u);
    return 2u * B * z + 32u * col_swizzle<B>(z) + 8u * (lane & 3u);
}

template <int OFF>
__device__ __forceinline__ u32x2_t ds_read_tr(uint32_t addr) {
    u32x2_t v;
    asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "i"(OFF));
    return v;
}

/* A subtile's fragments of a stage: the two halves of its 64 z. */
template <bool COLS>
struct Fragment;
template <>
struct Fragment<false> {
    u32x4_t v[2];
    __device__ __forceinline__ void ready() { after_wait(v[0]), after_wait(v[1]); }
    __device__ __forceinline__ bf16x8 operator[](int h) const { return __builtin_bit_cast(bf16x8, v[h]); }
};
template <>
struct Fragment<true> {
    u32x2_t v[2][2];
    __device__ __forceinline__ void ready() {
        after_wait(v[0][0]), after_wait(v[0][1]), after_wait(v[1][0]), after_wait(v[1][1]);
    }
    __device__ __forceinline__ bf16x8 operator[](int h) const {
        return __builtin_bit_cast(bf16x8, u32x4_t{v[h][0].x, v[h][0].y, v[h][1].x, v[h][1].y});
    }
};

template <class C>
struct TileRun {
    /* Load q of stage s is from at[q], in p or q moved on by s strides (of q 128 bytes), in an
     * extent of so many bytes. Operands of rows: of z, which lies inside them, those below Z;
     * p_z and q_z are an even q's, ^ 32 an odd one's. */
    const uint8_t *p_base, *q_base;
    uint64_t p_bytes, q_bytes, p_stride;
    uint32_t p_at[C::DA], q_at[C::DB], p_z, q_z, Z;
    uint32_t stages, wave, lane, wn, wt;

    __device__ __forceinline__ TileRun() {
        lane = threadIdx.x & 63u;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        wn = wave % C::WN, wt = wave / C::WN;
    }

    template <int Q>
    __device__ __forceinline__ void fetch_one(uint8_t *smem, uint32_t s, uint32_t slot) const {
        uint8_t *st = smem + C::STAGE * slot;
        const uint32_t now = min(s, stages - 1u); /* past the end the last stage again: the waits count */
        if constexpr (Q < C::DA) {
            /* of columns, the reduction's end is the range's */
            const Range r(p_base + p_stride * now, C::PCOLS ? p_bytes - p_stride * now : p_bytes);
            const bool in = C::PCOLS || kDepth * now + (p_z ^ 32u * (Q & 1)) < Z;
            r.template load<16>(in ? p_at[Q] : kNowhere, st + 1024u * (C::DA * wave + Q));
        } else {
            constexpr int q = Q - C::DA;
            const Range r(q_base + 2u * kDepth * now, q_bytes);
            const bool in = kDepth * now + (q_z ^ 32u * (C::DB > 1 ? q & 1 : 0)) < Z;
            r.template load<16>(in ? q_at[q] : kNowhere, st + C::A + 1024u * C::b_chunk(wave, q));
        }
    }
    template <int FROM, int TO>
    __device__ __forceinline__ void fetch(uint8_t *smem, uint32_t s, uint32_t slot) const {
        static_for<TO - FROM>([&](auto Q) { fetch_one<FROM + decltype(Q)::value>(smem, s, slot); });
    }

    /*
     * acc[j] += the products over all stages, for the first TL subtiles of a wave. Step
     * s, subtile j: the reads of subtile j + 1, the wait for those of j, eight
     * products. Before the last subtile's products the stage's LDS has been read by
     * this wave; behind a barrier there (all waves have, and stage s + 1 has landed
     * for all) its products run over the reads of the next stage's first fragments.
     */
    template <int TL>
    __device__ __forceinline__ void run(f32x4 (&acc)[C::TI][4], uint8_t *smem) {
        const uint32_t g = lane >> 4, c = lane & 15u;
        const uint32_t base = lds_addr(smem), lo = a_slot(c, g), hi = a_slot(c, 4u + g);
        uint32_t p_lo, p_hi = 0u;
        if constexpr (C::PCOLS)
            p_lo = base + (col_slot<C::BP>(lane) ^ 128u * wn);
        else
            p_lo = base + 8192u * wn + lo, p_hi = base + 8192u * wn + hi;
        const uint32_t q_lo = base + C::A + 2048u * wt + lo, q_hi = base + C::A + 2048u * wt + hi;
        Fragment<C::PCOLS> pf[4];
        Fragment<false> qf[2];
        uint32_t st = 0u;
        auto read_p = [&](auto I, auto H) {
            constexpr int i = decltype(I)::value, h = decltype(H)::value;
            if constexpr (C::PCOLS) {
                const uint32_t a = (p_lo + st) ^ (32u * i);
                pf[i].v[h][0] = ds_read_tr<(int)C::BP * 64 * h>(a);
                pf[i].v[h][1] = ds_read_tr<(int)C::BP * (64 * h + 8)>(a);
            } else {
                pf[i].v[h] = ds_read16<2048 * i>((h ? p_hi : p_lo) + st);
            }
        };
        auto read_q = [&](auto J) {
            constexpr int j = decltype(J)::value;
            qf[j & 1].v[0] = ds_read16<4096 * j>(q_lo + st);
            qf[j & 1].v[1] = ds_read16<4096 * j>(q_hi + st);
        };
        auto barrier = [] {
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        };
#pragma unroll
        for (int s = 0; s < C::STAGES - 1; s++) fetch<0, C::D>(smem, (uint32_t)s, (uint32_t)s);
        if constexpr (C::EARLY) fetch<0, C::DA + C::HALF>(smem, 1u, 1u);
        wait_vm<C::EARLY ? C::DA + C::HALF : C::D *(C::STAGES - 2)>();
        barrier();
        static_for<4>([&](auto I) {
            read_p(I, std::integral_constant<int, 0>{});
            read_p(I, std::integral_constant<int, 1>{});
        });
        read_q(std::integral_constant<int, 0>{});
        uint32_t slot = 0u, next = C::STAGES - 1;
        for (uint32_t s = 0; s < stages; s++) {
            const uint32_t ahead = s + C::STAGES - 1u, to = next;
            if constexpr (TL == 1) fetch<0, C::D>(smem, ahead, to);
            next = slot;
            slot = slot + 1u == (uint32_t)C::STAGES ? 0u : slot + 1u;
            static_for<TL>([&](auto J) {
                constexpr int j = decltype(J)::value;
                constexpr bool last = j + 1 == TL;
                if constexpr (!last) read_q(std::integral_constant<int, j + 1>{});
                wait_lgkm<last ? 0 : 2>(); /* the next subtile's reads stay out */
                if constexpr (j == 0) static_for<4>([&](auto I) { pf[decltype(I)::value].ready(); });
                qf[j & 1].ready();
                if constexpr (last) {
                    /* this wave's loads of stage s + 1; later ones stay out */
                    wait_vm<!C::EARLY ? C::D *(C::STAGES - 2) : TL == 4 ? 0 : C::DA + C::HALF>();
                    barrier();
                    st = C::STAGE * slot;
                }
                static_for<2>([&](auto H) {
                    constexpr int h = decltype(H)::value;
                    static_for<4>([&](auto I) {
                        constexpr int i = decltype(I)::value;
                        acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pf[i][h], qf[j & 1][h],
                                                                            acc[j][i], 0, 0, 0);
                        if constexpr (last) read_p(I, H);
                        __builtin_amdgcn_sched_barrier(0);
                        /* the loads ahead, spread over the products before the last
                         * subtile's: at once they would keep the waves from their reads */
                        constexpr int at = 8 * j + 4 * h + i;
                        if constexpr (TL == 1) {
                        } else if constexpr (C::EARLY) {
                            /* four subtiles: the stage's end is the second barrier */
                            constexpr int mid = 25, end = TL == 4 ? 32 : 8 * (TL - 1);
                            static_for<C::DB - C::HALF>([&](auto Q) {
                                constexpr int q = decltype(Q)::value;
                                if constexpr (q * 24 / (C::DB - C::HALF) == at)
                                    fetch_one<C::DA + C::HALF + q>(smem, ahead, to);
                            });
                            if constexpr (at == mid && TL != 4) barrier();
                            static_for<C::DA + C::HALF>([&](auto Q) {
                                constexpr int q = decltype(Q)::value;
                                if constexpr (mid + q * (end - mid) / (C::DA + C::HALF) == at)
                                    fetch_one<q>(smem, s + 2u, to ^ 1u);
                            });
                        } else {
                            constexpr int half = 8 * ((TL + 1) / 2);
                            static_for<C::D>([&](auto Q) {
                                if constexpr (decltype(Q)::value * half / C::D == at)
                                    fetch_one<decltype(Q)::value>(smem, ahead, to);
                            });
                        }
                    });
                });
                if constexpr (last) read_q(std::integral_constant<int, 0>{});
            });
        }
        wait_lgkm<0>(); /* the reads past the end: their registers stay taken till here */
        static_for<4>([&](auto I) { pf[decltype(I)::value].ready(); });
        qf[0].ready();
        wait_vm<0>(); /* the loads past the end land before the LDS is used again */
    }
};

template <class C>
__device__ __forceinline__ void run_steps(TileRun<C> &R, f32x4 (&acc)[C::TI][4], uint8_t *smem,
                                          uint32_t count) {
#pragma unroll
    for (int j = 0; j < C::TI; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[j][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (R.stages == 0u) return;
    /* a loop for each number of 32-row steps from TI / 2 on: fewer steps take that one,
     * with the last row in the place of those it has not */
    const uint32_t steps = (count + 31u) / 32u;
    bool done = false;
    static_for<C::TI / 2>([&](auto Q) {
        constexpr int tl = C::TI / 2 + decltype(Q)::value;
        if (!done && steps <= (uint32_t)tl) {
            R.template run<tl>(acc, smem);
            done = true;
        }
    });
    if (!done) R.template run<C::TI>(acc, smem);
}

/* One row tile x 64 WN columns of a product or an input gradient. */
template <class C, uint32_t LDS>
__device__ __forceinline__ void row_tile(const GroupArgs &A, uint8_t *smem, const RowTile &t,
                                         uint32_t col) {
    static_assert(C::LDS <= LDS && 2u * C::BP * C::BQ + 4u * C::BQ <= LDS, "stages; tile and rows");
    TileRun<C> R;
    const uint32_t L = R.lane, p0 = C::BP * col;
    R.stages = (A.Z + kDepth - 1u) / kDepth, R.Z = A.Z;
    /* W[z, p] or W[p, z] */
    const uint64_t first = C::PCOLS ? p0 : (uint64_t)p0 * A.Z, all = (uint64_t)A.P * A.Z;
    R.p_stride = 2u * kDepth * (C::PCOLS ? (uint64_t)A.P : 1u);
    R.p_base = (const uint8_t *)(A.p + t.expert * all + first);
    R.p_bytes = 2u * (all - first);
    R.p_z = 8u * a_dma_piece(L, 0u);
#pragma unroll
    for (int q = 0; q < C::DA; q++) {
        const uint32_t ch = C::DA * R.wave + (uint32_t)q;
        if constexpr (C::PCOLS) {
            const uint32_t piece = col_dma_piece<C::BP>(L, ch);
            R.p_at[q] = 2u * (col_dma_z<C::BP>(L, ch) * A.P + min(8u * piece, A.P - 8u - p0));
        } else {
            const uint32_t h = ch & 1u, r = min(16u * (ch >> 1) + a_dma_row(L, h), A.P - 1u - p0);
            R.p_at[q] = 2u * (r * A.Z + 8u * a_dma_piece(L, h));
        }
    }
    R.q_base = (const uint8_t *)(A.q_index ? A.q : A.q + (uint64_t)t.row * A.Z);
    R.q_bytes = 2u * (uint64_t)(A.q_index ? A.q_rows : t.rows) * A.Z;
    R.q_z = 8u * a_dma_piece(L, C::b_chunk(R.wave, 0u) & 1u);
#pragma unroll
    for (int q = 0; q < C::DB; q++) {
        const uint32_t ch = C::b_chunk(R.wave, (uint32_t)q), h = ch & 1u;
        uint32_t r = min(16u * (ch >> 1) + a_dma_row(L, h), t.rows - 1u);
        if (A.q_index) r = A.q_index[t.row + r];
        R.q_at[q] = !A.q_index || r < A.q_rows ? 2u * (r * A.Z + 8u * a_dma_piece(L, h)) : kNowhere;
    }
    f32x4 acc[C::TI][4];
    run_steps<C>(R, acc, smem, t.rows);
    /* the tile goes through LDS, 2 BP bytes a row, and leaves in 16-byte pieces of
     * whole rows; piece p of row r lies at p ^ r modulo their number */
    const uint32_t g = L >> 4, c = L & 15u;
    constexpr uint32_t PIECES = C::BP / 8u;
    /* read here once: a load in the loop of stores would wait for each */
    uint32_t *const rows = (uint32_t *)(smem + 2u * C::BP * C::BQ);
    uint32_t mine = ~0u;
    if (threadIdx.x < t.rows) {
        mine = t.row + threadIdx.x;
        if (A.to) {
            mine = A.to[mine];
            if (mine >= A.to_rows) mine = ~0u;
        }
    }
    __syncthreads();
    static_for<C::TI>([&](auto J) {
        constexpr int j = decltype(J)::value;
        if (32u * j >= t.rows) return;
        const uint32_t r = 16u * (2u * j + R.wt) + c;
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++) {
            const uint32_t p = 8u * R.wn + 2u * i + (g >> 1);
            *(uint2 *)(smem + 16u * (PIECES * r + (p ^ (r & (PIECES - 1u)))) + 8u * (g & 1u)) =
                bf16x4(acc[j][i]);
        }
    });
    if (threadIdx.x < C::BQ) rows[threadIdx.x] = mine;
    __syncthreads();
    const uint32_t width = min(C::BP, A.P - p0); /* a multiple of 8 */
    const uint32_t p = threadIdx.x % PIECES;
    if (8u * p >= width) return;
    /* Whole lines pass the caches by. us, as usual stores and so, products of 4096 tokens: 1024 x 2048,
     * 4 of 64 experts, 108 and 98, 2048 x 512 54 and 51, 4096 x 7168, 8 of 32, 1512 and 1530 (1000
     * tokens 513 and 499); forward and backward of a layer, one after the other, level. Rows that end
     * inside a line: 1040 x 1096, 3 of 24, 56 either way. */
    const auto store = [&](auto nontemporal) {
        for (uint32_t r = threadIdx.x / PIECES; r < t.rows; r += C::THREADS / PIECES) {
            const uint32_t to = rows[r];
            if (to == ~0u) continue;
            const u32x4_t v = *(const u32x4_t *)(smem + 16u * (PIECES * r + (p ^ (r & (PIECES - 1u)))));
            u32x4_t *place = (u32x4_t *)((uint16_t *)A.out + (uint64_t)to * A.P + p0 + 8u * p);
            if constexpr (decltype(nontemporal)::value) __builtin_nontemporal_store(v, place);
            else *place = v;
        }
    };
    if (A.P % 64u == 0u) store(std::true_type{});
    else store(std::false_type{});
}

/*
 * Tiles of 64 WN columns. A block's class goes by the rows of its expert: a CU holds one block
 * of any, so the largest's registers and LDS cost the others nothing. With few rows an expert bound by the
 * weights, read once: 488 rows of 32 experts of 7168 x 2048 170 us, 5.5 TB/s (a large read 6.1). With
 * many by the matrix units and what feeds them: 32768 rows of 4096 x 7168 1570 us, 1.23 PFLOP/s (a large
 * library product 1.45), the input gradient of 7168 x 2048 830 us, 1.16 (medians of forty calls once the
 * clock has settled; the least 1505 and 807). A stage of 256 x 256 takes 1.14
 * us with its operands in L2, 1.37 from memory, and 1.01 of matrix instructions alone; more stages,
 * blocks that stay and load their next tile ahead (1690 us), other orders and staggered starts measured
 * level or slower.
 */
template <int DIR, int WN>
__global__ __launch_bounds__(128 * WN, WN / 2) void grouped_rows_kernel(GroupArgs A) {
    using Tile32 = Tile<DIR, WN, 1, 4>;
    using Tile64 = Tile<DIR, WN, 2, 3>;
    using Tile128 = Tile<DIR, WN, 4, 3>;
    using Tile256 = Tile<DIR, WN, 8, 2>;
    constexpr uint32_t LDS = Tile128::LDS;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[LDS];
    RowTile t;
    uint32_t col;
    if (!find_tile<256u>(A, blockIdx.x, t, col)) return;
    if (t.n <= 32u) row_tile<Tile32, LDS>(A, smem, t, col);
    else if (t.n <= 64u) row_tile<Tile64, LDS>(A, smem, t, col);
    else if (t.n <= 128u) row_tile<Tile128, LDS>(A, smem, t, col);
    else row_tile<Tile256, LDS>(A, smem, t, col);
}

/*
 * A product of few rows: up to 16 of an expert x 16 of p a block, whose eight waves share z: pairs
 * of 32, so that a wave reads whole 128-byte lines, straight into the registers of the MFMA
 * layout, and add up through LDS in one order. More blocks than tiles of 256 p, and
 * no stage to fill: bound by the latency of two loads, then by the weights' stream. 4 rows of 4 of 64
 * experts of 1024 x 2048 5.9 us (5.3 from the caches), of which their 16.8 MB take 2.8 at 6.1 TB/s.
 */
__global__ __launch_bounds__(512) void grouped_few_kernel(GroupArgs A) {
    __shared__ f32x4 sums[8][64];
    RowTile t;
    uint32_t col;
    if (!find_tile<16u>(A, blockIdx.x, t, col)) return;
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, c = lane & 15u, n0 = 16u * col;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint16_t *w = A.p + (uint64_t)t.expert * A.P * A.Z + (uint64_t)min(n0 + c, A.P - 1u) * A.Z;
    uint32_t r = t.row + min(c, t.rows - 1u), to = r;
    if (A.to) to = A.to[r];
    bool row = true;
    if (A.q_index) {
        r = A.q_index[r];
        row = r < A.q_rows;
    }
    const uint16_t *x = A.q + (uint64_t)(row ? r : 0u) * A.Z;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int DEEP = 4; /* pairs under way */
    for (uint32_t k = 64u * wave; k < A.Z; k += 512u * DEEP) {
        u32x4_t a[DEEP][2], b[DEEP][2];
#pragma unroll
        for (int i = 0; i < DEEP; i++)
#pragma unroll
            for (uint32_t h = 0; h < 2u; h++) {
                const uint32_t z = k + 512u * (uint32_t)i + 32u * h + 8u * g;
                a[i][h] = b[i][h] = u32x4_t{0u, 0u, 0u, 0u};
                if (z < A.Z) { /* 8 of z, a multiple of 8 */
                    a[i][h] = __builtin_nontemporal_load((const u32x4_t *)(w + z));
                    if (row) b[i][h] = *(const u32x4_t *)(x + z);
                }
            }
#pragma unroll
        for (int i = 0; i < DEEP; i++)
#pragma unroll
            for (int h = 0; h < 2; h++)
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[i][h]),
                                                              __builtin_bit_cast(bf16x8, b[i][h]), acc, 0, 0, 0);
    }
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave != 0u) return;
#pragma unroll
    for (int v = 1; v < 8; v++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[i] = __fadd_rn(acc[i], sums[v][lane][i]);
    if (c < t.rows && n0 + 4u * g < A.P && (!A.to || to < A.to_rows))
        *(uint2 *)((uint16_t *)A.out + (uint64_t)to * A.P + n0 + 4u * g) = bf16x4(acc);
}

/* ---------------------------------------------------------------------- */
/* weight gradient                                                         */
/* ---------------------------------------------------------------------- */

/*
 * A block holds 128 of p (columns of x) x 256 of q (columns of dy), in four waves of 64 x 128,
 * and two blocks lie on a CU: a reduction is as long as an expert has rows, often only a few
 * stages, and one block's first loads and its stores (128 KB in f32) run under the other's products.
 * A stage is 32 rows; q is kept as two panels of 128 columns. 4000 rows of 64 experts of 2048 x 512
 * to bf16 32 us, 27 of which the 147 MB take as a large copy; 32768 rows of 32 experts of 4096 x 7168 to
 * f32 2060 to 2200 us by the card, 0.87 to 0.93 PFLOP/s (a large library product of such
 * operands 1.18), to bf16 1850. Bound by power, operands and the stages' own waits: of the last, on
 * zeros 1540 (the clock falls less), with the operands in L2 1610, with both 1265. Waves of 128 x 128, four of
 * them and 256 x 256 a block, read a third less of LDS, but one wave a SIMD has its 250 instructions a
 * stage to issue by itself and leaves its waits and stores bare: 1915, on zeros 1830; 1000 tokens 790
 * and 645, 64 experts of 1024 x 2048 83 and 60.
 */
struct Weight {
    static constexpr uint32_t BP = 128, BQ = 256, DEPTH = 32, STAGES = 3, WAVES = 4, THREADS = 256;
    static constexpr uint32_t A = BP * DEPTH * 2, B = BQ * DEPTH * 2, STAGE = A + B, PANEL = B / 2;
    static constexpr int DA = 2, DB = 4, D = DA + DB; /* loads of 1 KB, four rows of 128 columns, a wave */
    static constexpr int TI = 8;                      /* subtiles of q of a wave */
};

/*
 * The rows that an operand picks by an index. A wave loads rows 8 wave .. + 8 of a stage; their
 * indices come through LDS as well, by a load of its own that the waits count like any other (one
 * to registers the compiler would wait for with all others out), into a ring of stages.
 */
struct Picks {
    static constexpr uint32_t kRing = 4, SLOT = 256, BYTES = SLOT * kRing; /* a load fills a slot */
    const uint32_t *index; /* from the expert's first row on; NULL: rows as they lie, nothing is read */
    uint32_t rows, at;     /* at: this lane's place among the indices of a stage */
    uint8_t *held;         /* this wave's */

    __device__ __forceinline__ void fetch(uint32_t now, uint32_t slot) const {
        Range(index + Weight::DEPTH * now, index ? 4u * (uint64_t)(rows - Weight::DEPTH * now) : 0u)
            .load<4>(at, held + SLOT * slot);
    }
    /* The places of this lane's two rows of a stage by the indices read: its row times the row's
     * bytes. Rows past the expert's last, or the tensor's, lie past the range's end. The products
     * are of 24 bits: a row of up to 65535, its bytes. */
    __device__ __forceinline__ uint32_t place(uint32_t read, uint32_t now, uint32_t z, uint32_t row_bytes) const {
        const bool live = Weight::DEPTH * now + z < rows;
        return __umul24(index ? live ? min(read, kMostPicked) : kMostPicked : z, row_bytes);
    }
};

struct WeightRun {
    using C = Weight;
    const uint8_t *p_base, *q_base; /* moved on by a stride each stage where rows lie in order */
    uint64_t p_bytes, q_bytes, p_stride, q_stride;
    Picks p, q;
    uint32_t p_row_bytes, q_row_bytes, p_col[2], q_col[4]; /* the loads' columns */
    uint32_t p_at[2], q_at[2];                             /* and rows, of the stage that is loaded */
    uint32_t stages, wave, lane, wn, wt;

    __device__ __forceinline__ WeightRun() {
        lane = threadIdx.x & 63u;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        wn = wave % 2u, wt = wave / 2u;
    }
    __device__ __forceinline__ uint32_t clamped(uint32_t s) const { return min(s, stages - 1u); }
    __device__ __forceinline__ void fetch_picks(uint32_t s) const {
        p.fetch(clamped(s), s % Picks::kRing);
        q.fetch(clamped(s), s % Picks::kRing);
    }
    __device__ __forceinline__ void read_picks(uint32_t s, uint32_t (&r)[4]) const {
        const uint32_t at = Picks::SLOT * (s % Picks::kRing) + 4u * (lane >> 4);
        r[0] = ds_read4<0>(lds_addr(p.held) + at), r[1] = ds_read4<16>(lds_addr(p.held) + at);
        r[2] = ds_read4<0>(lds_addr(q.held) + at), r[3] = ds_read4<16>(lds_addr(q.held) + at);
    }
    __device__ __forceinline__ void set_rows(uint32_t s, uint32_t (&r)[4]) {
        static_for<4>([&](auto I) { after_wait(r[decltype(I)::value]); });
        const uint32_t now = clamped(s), z = 8u * wave + (lane >> 4);
        p_at[0] = p.place(r[0], now, z, p_row_bytes), p_at[1] = p.place(r[1], now, z + 4u, p_row_bytes);
        q_at[0] = q.place(r[2], now, z, q_row_bytes), q_at[1] = q.place(r[3], now, z + 4u, q_row_bytes);
    }
    /* Load Q of stage s; past the end the last stage again, so that the counts of the waits stay. */
    template <int Q>
    __device__ __forceinline__ void fetch_one(uint8_t *smem, uint32_t s, uint32_t slot) const {
        uint8_t *st = smem + C::STAGE * slot;
        const uint32_t now = clamped(s);
        if constexpr (Q < C::DA) {
            Range(p_base + p_stride * now, p_bytes - p_stride * now)
                .load<16>(p_at[Q] + p_col[Q], st + 1024u * (2u * wave + Q));
        } else {
            constexpr int q = Q - C::DA;
            Range(q_base + q_stride * now, q_bytes - q_stride * now)
                .load<16>(q_at[q & 1] + q_col[q], st + C::A + C::PANEL * (q >> 1) + 1024u * (2u * wave + (q & 1)));
        }
    }
    /* Loads FROM .. TO of a stage to its slot, s < 3; and of the first two. */
    template <int FROM, int TO>
    __device__ __forceinline__ void fetch_stage(uint8_t *smem, uint32_t s) const {
        static_for<TO - FROM>([&](auto Q) { fetch_one<FROM + decltype(Q)::value>(smem, s, s); });
    }
    template <int FROM, int TO>
    __device__ __forceinline__ void fetch(uint8_t *smem) const {
        fetch_stage<FROM, TO>(smem, 0u);
        fetch_stage<FROM, TO>(smem, 1u);
    }

    /* acc[j] += the products over all stages, for the first 2 PAIRS subtiles of a wave, two a step, as
     * in TileRun: a step's reads run under the products of the one before. */
    template <int PAIRS>
    __device__ __forceinline__ void run(f32x4 (&acc)[C::TI][4], uint8_t *smem) {
        const uint32_t base = lds_addr(smem);
        const uint32_t p_lo = base + (col_slot<128u>(lane) ^ 128u * wn);
        const uint32_t q_lo = base + C::A + (col_slot<128u>(lane) ^ 32u * wt);
        u32x2_t pf[4][2], qf[2][2][2];
        uint32_t st = 0u;
        auto read_p = [&](auto I) {
            constexpr int i = decltype(I)::value;
            const uint32_t a = (p_lo + st) ^ (32u * i);
            pf[i][0] = ds_read_tr<0>(a), pf[i][1] = ds_read_tr<1024>(a);
        };
        auto read_q = [&](auto S) {
            constexpr int step = decltype(S)::value;
            static_for<2>([&](auto J) {
                constexpr int j = 2 * step + decltype(J)::value, panel = C::PANEL * (j >> 2);
                const uint32_t a = (q_lo + st) ^ (64u * (j & 3));
                qf[step & 1][j & 1][0] = ds_read_tr<panel>(a), qf[step & 1][j & 1][1] = ds_read_tr<panel + 1024>(a);
            });
        };
        auto whole = [](const u32x2_t (&v)[2]) {
            return __builtin_bit_cast(bf16x8, u32x4_t{v[0].x, v[0].y, v[1].x, v[1].y});
        };
        auto barrier = [] {
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        };
        /* the first stages of an operand whose rows lie in order are under way while the other's
         * indices are waited for */
        uint32_t next_rows[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (uint32_t s = 0; s < 3u; s++) fetch_picks(s);
        set_rows(0u, next_rows);
        if (!p.index) fetch<0, C::DA>(smem);
        if (!q.index) fetch<C::DA, C::D>(smem);
        if (p.index || q.index) {
            if (!q.index) wait_vm<2 * C::DB>();
            else if (!p.index) wait_vm<2 * C::DA>();
            else wait_vm<0>();
            uint32_t rows[2][4];
            read_picks(0u, rows[0]);
            read_picks(1u, rows[1]);
            wait_lgkm<0>();
            static_for<2>([&](auto S) {
                constexpr uint32_t s = decltype(S)::value;
                set_rows(s, rows[s]);
                if (p.index) fetch_stage<0, C::DA>(smem, s);
                if (q.index) fetch_stage<C::DA, C::D>(smem, s);
            });
        }
        wait_vm<0>(); /* stages 0 and 1, which came close behind it */
        barrier();
        static_for<4>(read_p);
        read_q(std::integral_constant<int, 0>{});
        uint32_t slot = 0u, to = 2u;
        for (uint32_t s = 0; s < stages; s++) {
            /* stage s + 2's rows have landed, s + 3's are loaded ahead of the rest */
            read_picks(s + 2u, next_rows);
            fetch_picks(s + 3u);
            const uint32_t free = to;
            to = slot;
            slot = slot + 1u == C::STAGES ? 0u : slot + 1u;
            static_for<PAIRS>([&](auto S) {
                constexpr int step = decltype(S)::value;
                constexpr bool last = step + 1 == PAIRS;
                if constexpr (!last) read_q(std::integral_constant<int, step + 1>{});
                wait_lgkm<last ? 0 : 4>();
                if constexpr (step == 0) {
                    static_for<4>([&](auto I) {
                        after_wait(pf[decltype(I)::value][0]);
                        after_wait(pf[decltype(I)::value][1]);
                    });
                    set_rows(s + 2u, next_rows);
                }
                static_for<2>([&](auto J) {
                    after_wait(qf[step & 1][decltype(J)::value][0]);
                    after_wait(qf[step & 1][decltype(J)::value][1]);
                });
                if constexpr (last) {
                    wait_vm<C::D>(); /* stage s + 1 has landed; this stage's loads stay out */
                    barrier();
                    st = C::STAGE * slot;
                }
                static_for<2>([&](auto J) {
                    constexpr int j = 2 * step + decltype(J)::value;
                    static_for<4>([&](auto I) {
                        constexpr int i = decltype(I)::value;
                        acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(whole(pf[i]), whole(qf[step & 1][j & 1]),
                                                                            acc[j][i], 0, 0, 0);
                        if constexpr (last && (j & 1) == 1) read_p(I);
                        __builtin_amdgcn_sched_barrier(0);
                        /* the loads ahead, spread over the steps before the last */
                        constexpr int at = 4 * j + i;
                        static_for<C::D>([&](auto Q) {
                            if constexpr (1 + decltype(Q)::value * (8 * (PAIRS - 1) - 1) / C::D == at)
                                fetch_one<decltype(Q)::value>(smem, s + 2u, free);
                        });
                    });
                });
                if constexpr (last) read_q(std::integral_constant<int, 0>{});
            });
        }
        wait_lgkm<0>(); /* the reads past the end: their registers stay taken till here */
        static_for<4>([&](auto I) {
            after_wait(pf[decltype(I)::value][0]);
            after_wait(pf[decltype(I)::value][1]);
        });
        static_for<2>([&](auto J) {
            after_wait(qf[0][decltype(J)::value][0]);
            after_wait(qf[0][decltype(J)::value][1]);
        });
        wait_vm<0>(); /* the loads past the end land before the LDS is used again */
    }
};

/* XCD x (blocks x, x + 8, ...; it has an L2 of its own) takes runs of 16 tiles, which share operands, and
 * the XCDs take the runs in turn, so that experts with many rows fall to all of them. us, in one
 * contiguous range an XCD and so: 4096 tokens, 8 of 32 experts of 4096 x 7168 (bf16), rows spread evenly
 * 1925 and 1945, by a skewed router 2279 and 1948; 1000 tokens, 4 of 64 of 1024 x 2048, 70 and
 * 65, skewed 78 and 68 (runs of 64 tiles 71 and 84, of 4 66 and 66). */
constexpr uint32_t kRun = 16;

template <bool F32>
__global__ __launch_bounds__(256, 2) void grouped_weight_kernel(GroupArgs A) {
    using C = Weight;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[C::STAGES * C::STAGE];
    __shared__ uint8_t held[2][C::WAVES][Picks::BYTES];
    const uint32_t turn = blockIdx.x >> 3;
    uint32_t w = (turn / kRun * 8u + (blockIdx.x & 7u)) * kRun + turn % kRun;
    if (w >= A.E * A.tiles_p * A.tiles_q) return;
    const uint32_t expert = w / (A.tiles_p * A.tiles_q);
    w %= A.tiles_p * A.tiles_q;
    /* four q tiles at a time, along p */
    const uint32_t grp = w / (4u * A.tiles_p), in = w % (4u * A.tiles_p);
    const uint32_t many = min(4u, A.tiles_q - 4u * grp);
    const uint32_t p0 = C::BP * (in / many), q0 = C::BQ * (4u * grp + in % many);
    WeightRun R;
    const uint32_t L = R.lane, at = L < 8u ? 4u * (8u * R.wave + L) : kNowhere;
    uint32_t row;
    const uint32_t rows = rows_of(A.offsets, expert, A.R, row);
    R.stages = (rows + C::DEPTH - 1u) / C::DEPTH;
    R.p_row_bytes = 2u * A.P, R.q_row_bytes = 2u * A.Q;
    R.p = Picks{A.p_index ? A.p_index + row : nullptr, rows, at, held[0][R.wave]};
    R.q = Picks{A.q_index ? A.q_index + row : nullptr, rows, at, held[1][R.wave]};
    /* picked rows lie anywhere in the tensor, others move on with the stages */
    R.p_stride = A.p_index ? 0u : (uint64_t)C::DEPTH * R.p_row_bytes;
    R.q_stride = A.q_index ? 0u : (uint64_t)C::DEPTH * R.q_row_bytes;
    R.p_base = (const uint8_t *)(A.p + (A.p_index ? 0u : (uint64_t)row * A.P) + p0);
    R.q_base = (const uint8_t *)(A.q + (A.q_index ? 0u : (uint64_t)row * A.Q) + q0);
    R.p_bytes = (uint64_t)(A.p_index ? A.p_rows : rows) * R.p_row_bytes - 2u * p0;
    R.q_bytes = (uint64_t)(A.q_index ? A.q_rows : rows) * R.q_row_bytes - 2u * q0;
#pragma unroll
    for (uint32_t q = 0; q < 2u; q++) {
        const uint32_t col = 8u * col_dma_piece<128u>(L, 2u * R.wave + q);
        R.p_col[q] = 2u * min(col, A.P - 8u - p0);
        R.q_col[q] = 2u * min(col, A.Q - 8u - q0);
        R.q_col[2u + q] = 2u * min(128u + col, A.Q - 8u - q0);
    }
    const uint32_t high = min(C::BQ, A.Q - q0), width = min(C::BP, A.P - p0);
    f32x4 acc[C::TI][4];
#pragma unroll
    for (int j = 0; j < C::TI; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[j][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (R.stages != 0u) {
        if (high <= 128u) R.run<2>(acc, smem);
        else R.run<4>(acc, smem);
    }
    const uint32_t g = L >> 4, c = L & 15u;
    const uint64_t to = ((uint64_t)expert * A.Q + q0) * A.P + p0;
    /* Through LDS for stores of whole rows (64-byte pieces straight from the accumulators took 10 us for
     * 256 x 256): f32 128 rows at a time, bf16 all; piece p of row r lies at p ^ r modulo 16. The output
     * passes the caches by, which the operands are read from again. us, so and as usual stores: f32, 4096
     * tokens, 8 of 32 experts of 4096 x 7168, 2058 and 2204, 1000 tokens 814 and 1038, 4 of 16 of 4096
     * x 7176, 1000 tokens, 528 and 645; bf16 100, 1000 and 4096 tokens of the first 299 and 349, 590 and
     * 755, 1830 and 1885; but bf16 rows that end inside a 128-byte line are cut lines twice: 4 of 16
     * of 4096 x 7176, 100 tokens, 396 and 266 (1000 tokens 345 and 468), 3 of 24 of 1040 x 1096, 1000
     * tokens, 28.0 and 25.7. */
    constexpr uint32_t ROW = F32 ? 512u : 256u, HIGH = F32 ? 128u : 256u, PIECES = ROW / 16u;
    static_assert(ROW * HIGH <= sizeof smem, "the part of the tile");
    if (F32 && A.accumulate && R.stages == 0u) return;
    static_for<C::BQ / HIGH>([&](auto H) {
        constexpr int part = decltype(H)::value, JS = HIGH / 32;
        __syncthreads();
        static_for<JS>([&](auto J) {
            constexpr int j = decltype(J)::value;
            const uint32_t r = 16u * (2u * j + R.wt) + c;
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++) {
                const f32x4 &v = acc[JS * part + j][i];
                const uint32_t n = 16u * R.wn + 4u * i + g; /* of four columns */
                if constexpr (F32)
                    *(f32x4 *)(smem + ROW * r + 16u * (n ^ (r & 15u))) = v;
                else
                    *(uint2 *)(smem + ROW * r + 16u * (n >> 1 ^ (r & 15u)) + 8u * (n & 1u)) = bf16x4(v);
            }
        });
        __syncthreads();
        const uint32_t piece = threadIdx.x % PIECES;
        if ((F32 ? 4u : 8u) * piece >= width) return;
        const auto store = [&](auto nontemporal) {
#pragma unroll 4
            for (uint32_t r = threadIdx.x / PIECES; r < HIGH; r += C::THREADS / PIECES) {
                const uint32_t q = HIGH * part + r;
                if (q >= high) break;
                const u32x4_t v = *(const u32x4_t *)(smem + ROW * r + 16u * (piece ^ (r & 15u)));
                if constexpr (F32) {
                    f32x4 *place = (f32x4 *)((float *)A.out + to + (uint64_t)q * A.P + 4u * piece);
                    f32x4 sum = __builtin_bit_cast(f32x4, v);
                    if (A.accumulate) {
                        const f32x4 before = *place;
#pragma unroll
                        for (int k = 0; k < 4; k++) sum[k] = __fadd_rn(before[k], sum[k]);
                    }
                    __builtin_nontemporal_store(sum, place);
                } else {
                    u32x4_t *place = (u32x4_t *)((uint16_t *)A.out + to + (uint64_t)q * A.P + 8u * piece);
                    if constexpr (decltype(nontemporal)::value) __builtin_nontemporal_store(v, place);
                    else *place = v;
                }
            }
        };
        if (F32 || A.P % 64u == 0u) store(std::true_type{});
        else store(std::false_type{});
    });
}

/* ---------------------------------------------------------------------- */
/* host side                                                               */
/* ---------------------------------------------------------------------- */

bool sizes_ok(uint32_t rows, uint32_t experts, uint32_t N, uint32_t K) {
    return rows != 0u && rows <= kMostRows && experts != 0u && experts <= 1024u && N != 0u &&
           N % 8u == 0u && N <= kMostWidth && K != 0u && K % 8u == 0u && K <= kMostWidth;
}
bool aligned(const void *p, uintptr_t to) { return p && (uintptr_t)p % to == 0u; }

/* Rows of `have`, of which an index (nullable) picks `rows`. */
bool picks_ok(const uint32_t *index, uint32_t have, uint32_t rows) {
    return (uintptr_t)index % 4u == 0u && (index ? have != 0u && have <= kMostPicked : have >= rows);
}

/* Whether an output lies over the offsets or an index, which tiles read while others write. */
bool over_plan(const void *output, uint64_t bytes, const uint32_t *offsets, uint32_t experts,
               const uint32_t *index, const uint32_t *other, uint32_t rows) {
    return overlap(output, bytes, offsets, 4u * (uint64_t)(experts + 1u)) ||
           (index && overlap(output, bytes, index, 4u * (uint64_t)rows)) ||
           (other && overlap(output, bytes, other, 4u * (uint64_t)rows));
}

/* Most blocks of a product that goes 16 rows x 16 columns a block. us, weights from memory, so, by tiles
 * of 128 columns (narrow_tiles: what these products get instead) and of 256; rows of experts chosen at random
 * of 64: 1024 x 2048, 4 rows (256 blocks) 5.9, 10.4 and 15.9, 8 rows (512) 9.0, 10.7 and 16.2, 16 rows
 * (1088) 15.6, 14.6 and 20.8, 32 rows (2176) 21.9, 21.2 and 29.1; 2048 x 512, 4 rows (512) 4.5, 5.2 and 6.9,
 * 8 rows (1024) 6.9, 5.9 and 7.1, 16 rows (2176) 10.8, 9.2 and 10.6; of 32, 7168 x 2048, 2 rows (896) 15.4,
 * 11.6 and 16.4. Past 512 blocks the tiles of 128 are ahead by up to a quarter. */
constexpr uint64_t kFewBlocks = 1024;

/* Tiles of 128 columns instead of 256, where these leave half of the CUs without one: `used`
 * experts have up to 128 rows each, if these are spread evenly, and so one row tile. us, weights from
 * memory, of 256 and of 128 columns (N x K): product of 1040 x 1096, 24 experts, 24 rows 23.4 and 14.2, 384 rows
 * 26.4 and 17.1, 3000 rows 35.9 and 26.3, but 6000 rows 40.8 and 52.7; its input gradient, 24 rows 16.9 and
 * 11.8, 3000 rows 29.2 and 22.9, 6000 rows 33.6 and 47.6; input gradient of 2048 x 512, 64 experts, 244 rows
 * 32.2 and 26.9, 8000 rows 48.9 and 38.6; with more tiles, product of 1024 x 1024, 40 experts (160), 64 rows
 * 16.6 and 14.5, 366 rows 18.6 and 21.9, 1500 rows 20.0 and 24.7, of 1024 x 2048, 64 experts (256), 64 rows 46.7
 * and 47.5, 244 rows 62.8 and 60.0. Weights that the caches hold give the same order. */
bool narrow_tiles(uint32_t used, uint32_t rows, uint32_t P) {
    return (uint64_t)used * ((P + 255u) / 256u) <= 128u && rows <= 128u * used;
}

template <int DIR>
bool launch_rows(void *output, const void *input, const void *weights, const uint32_t *offsets,
                 const uint32_t *input_index, const uint32_t *output_index, uint32_t rows,
                 uint32_t input_rows, uint32_t output_rows, uint32_t experts, uint32_t N, uint32_t K,
                 hipStream_t st) {
    const uint32_t P = DIR == kProduct ? N : K, Z = DIR == kProduct ? K : N;
    if (!sizes_ok(rows, experts, N, K) || !aligned(output, 16u) || !aligned(input, 16u) ||
        !aligned(weights, 16u) || !aligned(offsets, 4u) || !picks_ok(input_index, input_rows, rows) ||
        (uintptr_t)output_index % 4u != 0u || output_rows == 0u || output_rows > kMostRows ||
        (!output_index && output_rows < rows))
        return false;
    const uint64_t out = 2u * (uint64_t)output_rows * P;
    /* tiles read all of a row while others write */
    if (overlap(output, out, input, 2u * (uint64_t)input_rows * Z) ||
        overlap(output, out, weights, 2u * (uint64_t)experts * N * K) ||
        over_plan(output, out, offsets, experts, input_index, output_index, rows))
        return false;
    GroupArgs A{};
    A.p = (const uint16_t *)weights, A.q = (const uint16_t *)input, A.offsets = offsets;
    A.q_index = input_index, A.to = output_index, A.q_rows = input_rows, A.to_rows = output_rows;
    A.out = output, A.R = rows, A.E = experts, A.P = P, A.Z = Z;
    /* n rows are in at most 1 + n / 16 tiles of 16, of experts that have rows */
    const uint32_t used = experts < rows ? experts : rows;
    const uint64_t few = (uint64_t)(rows / 16u + used) * ((P + 15u) / 16u);
    if (DIR == kProduct && few <= kFewBlocks) {
        A.tiles_p = (P + 15u) / 16u;
        hipLaunchKernelGGL(grouped_few_kernel, dim3((uint32_t)few + 8u), dim3(512), 0, st, A);
        return hipGetLastError() == hipSuccess;
    }
    const uint64_t tiles = rows / 256u + used;
    const bool narrow = narrow_tiles(used, rows, P);
    A.tiles_p = narrow ? (P + 127u) / 128u : (P + 255u) / 256u;
    const uint64_t blocks = tiles * A.tiles_p + 8u;
    if (blocks >= 1u << 23) return false; /* 2^32 threads */
    if (narrow)
        hipLaunchKernelGGL(HIP_KERNEL_NAME(grouped_rows_kernel<DIR, 2>), dim3((uint32_t)blocks), dim3(256), 0, st, A);
    else
        hipLaunchKernelGGL(HIP_KERNEL_NAME(grouped_rows_kernel<DIR, 4>), dim3((uint32_t)blocks), dim3(512), 0, st, A);
    return hipGetLastError() == hipSuccess;
}

}  // namespace
}  // namespace k3

using namespace k3;

extern "C" bool k3_moe_grouped_product_bf16(void *output, const void *input, const void *weights,
                                            const uint32_t *offsets, const uint32_t *input_index,
                                            const uint32_t *output_index, uint32_t rows,
                                            uint32_t input_rows, uint32_t output_rows,
                                            uint32_t expert_count, uint32_t out_columns,
                                            uint32_t columns, void *stream) {
    return launch_rows<kProduct>(output, input, weights, offsets, input_index, output_index, rows, input_rows,
                                 output_rows, expert_count, out_columns, columns, (hipStream_t)stream);
}

extern "C" bool k3_moe_grouped_input_gradient_bf16(void *output, const void *output_gradient,
                                                   const void *weights, const uint32_t *offsets,
                                                   const uint32_t *gradient_index,
                                                   const uint32_t *output_index, uint32_t rows,
                                                   uint32_t gradient_rows, uint32_t output_rows,
                                                   uint32_t expert_count, uint32_t out_columns,
                                                   uint32_t columns, void *stream) {
    return launch_rows<kInput>(output, output_gradient, weights, offsets, gradient_index, output_index, rows,
                               gradient_rows, output_rows, expert_count, out_columns, columns,
                               (hipStream_t)stream);
}

extern "C" bool k3_moe_grouped_weight_gradient_bf16(void *output, bool f32, bool accumulate,
                                                    const void *output_gradient, const void *input,
                                                    const uint32_t *offsets,
                                                    const uint32_t *gradient_index,
                                                    const uint32_t *input_index, uint32_t rows,
                                                    uint32_t gradient_rows, uint32_t input_rows,
                                                    uint32_t expert_count, uint32_t out_columns,
                                                    uint32_t columns, void *stream) {
    if (!sizes_ok(rows, expert_count, out_columns, columns) || !aligned(output, 16u) ||
        !aligned(output_gradient, 16u) || !aligned(input, 16u) || !aligned(offsets, 4u) ||
        !picks_ok(gradient_index, gradient_rows, rows) || !picks_ok(input_index, input_rows, rows) ||
        (accumulate && !f32))
        return false;
    const uint64_t values = (uint64_t)expert_count * out_columns * columns, out = (f32 ? 4u : 2u) * values;
    if (overlap(output, out, output_gradient, 2u * (uint64_t)gradient_rows * out_columns) ||
        overlap(output, out, input, 2u * (uint64_t)input_rows * columns) ||
        over_plan(output, out, offsets, expert_count, gradient_index, input_index, rows))
        return false;
    GroupArgs A{};
    A.p = (const uint16_t *)input, A.q = (const uint16_t *)output_gradient, A.offsets = offsets;
    A.p_index = input_index, A.q_index = gradient_index, A.p_rows = input_rows, A.q_rows = gradient_rows;
    A.out = output, A.R = rows, A.E = expert_count, A.P = columns, A.Q = out_columns;
    A.accumulate = accumulate;
    A.tiles_p = (columns + Weight::BP - 1u) / Weight::BP, A.tiles_q = (out_columns + Weight::BQ - 1u) / Weight::BQ;
    const uint64_t all = 8u * kRun; /* whole turns of the XCDs */
    const uint64_t blocks = ((uint64_t)expert_count * A.tiles_p * A.tiles_q + all - 1u) / all * all;
    if (blocks >= 1u << 23) return false;
    const auto kernel = f32 ? grouped_weight_kernel<true> : grouped_weight_kernel<false>;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(Weight::THREADS), 0, (hipStream_t)stream, A);
    return hipGetLastError() == hipSuccess;
}
