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
 * bytes a lane; one of columns as 64 rows of z, and read by the transposing LDS
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

enum Direction { kProduct, kInput, kWeight };

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
    return make_uint2(f32_to_bf16(v[0]) | (uint32_t)f32_to_bf16(v[1]) << 16,
                      f32_to_bf16(v[2]) | (uint32_t)f32_to_bf16(v[3]) << 16);
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

__device__ __forceinline__ uint32_t tiles_of(uint32_t n) { return (n + 255u) / 256u; }

__device__ __forceinline__ uint32_t wave_scan(uint32_t v, uint32_t lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t a = __shfl_up(v, o, 64);
        if ((int)lane >= o) v += a;
    }
    return v;
}

struct RowTile {
    uint32_t expert, row, rows, many, index, n; /* n: the expert's rows, in `many` tiles */
};

/*
 * Row tile and column of work `block` among all experts' row tiles x tiles_p columns,
 * found by every wave for itself from the offsets: each lane counts the tiles of
 * up to 16 consecutive experts, and the lanes then take those of the one that holds the
 * tile. About 1 us, where a launch that lists the tiles takes 4. An expert's tiles
 * of one column are neighbours, as they read the same weights; XCD x (blocks x,
 * x + 8, ...) takes a contiguous range of the works. False past the end.
 */
__device__ __forceinline__ bool find_tile(const GroupArgs &A, uint32_t block, RowTile &t,
                                          uint32_t &col) {
    const uint32_t lane = threadIdx.x & 63u, per = (A.E + 63u) / 64u;
    uint32_t mine = 0u;
    for (uint32_t i = 0; i < per; i++) {
        const uint32_t e = lane * per + i;
        uint32_t begin;
        if (e < A.E) mine += tiles_of(rows_of(A.offsets, e, A.R, begin));
    }
    const uint32_t upto = wave_scan(mine, lane);
    const uint32_t total = __builtin_amdgcn_readlane(upto, 63);
    const uint32_t works = total * A.tiles_p, each = (works + 7u) / 8u;
    const uint32_t w = (block & 7u) * each + (block >> 3);
    if ((block >> 3) >= each || w >= works) return false;
    const uint32_t tile = w / A.tiles_p; /* an expert's tiles x columns, before its order is set */
    const uint32_t owner = __builtin_ctzll(__ballot(upto > tile));
    const uint32_t before = __builtin_amdgcn_readlane(upto - mine, owner);
    const uint32_t e = owner * per + lane;
    uint32_t begin = 0u, n = 0u;
    if (lane < per && e < A.E) n = rows_of(A.offsets, e, A.R, begin);
    const uint32_t many = tiles_of(n), to = before + wave_scan(many, lane);
    const uint32_t at = __builtin_ctzll(__ballot(to > tile));
    t.n = __builtin_amdgcn_readlane(n, at);
    t.many = __builtin_amdgcn_readlane(many, at);
    t.expert = owner * per + at;
    const uint32_t first = __builtin_amdgcn_readlane(to, at) - t.many;
    const uint32_t local = (tile - first) * A.tiles_p + w % A.tiles_p;
    const uint32_t height = tile_height(t.n);
    t.index = local % t.many;
    col = local / t.many;
    t.row = __builtin_amdgcn_readlane(begin, at) + height * t.index;
    t.rows = t.n > height * t.index ? min(height, t.n - height * t.index) : 0u;
    return true;
}

/* 64 WN of p x 32 TI of q a block of 2 WN waves; wave (wn, wt) holds p 64 wn .. + 64
 * and the subtiles (16 q) wt, wt + 2, ... */
template <int DIR_, int WN_, int TI_, int STAGES_>
struct Tile {
    static constexpr int DIR = DIR_, WN = WN_, TI = TI_, STAGES = STAGES_, WAVES = 2 * WN,
                         THREADS = 64 * WAVES;
    static constexpr bool PCOLS = DIR != kProduct, QCOLS = DIR == kWeight;
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
    static_assert(!EARLY || (TI == 8 && WAVES == 8), "two panels of 128 q");
    static constexpr int HALF = EARLY ? DB / 2 : 0; /* loads of the first panel */
    static constexpr int QREADS = QCOLS ? 4 : 2;    /* of a subtile */
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

/*
 * The rows that an operand of a weight gradient picks by an index. A wave loads z = 8 wave .. + 8
 * of a stage; their indices come through LDS as well, by a load of its own that the waits
 * count like any other (one to registers the compiler would wait for with all others out),
 * into a ring of stages.
 */
struct Picks {
    static constexpr uint32_t kRing = 4, SLOT = 256, BYTES = SLOT * kRing; /* a load fills a slot */
    const uint32_t *index; /* from the tile's first row on; NULL: rows as they lie, nothing is read */
    uint32_t rows, at;     /* at: this lane's place among the indices of a stage */
    uint8_t *held;         /* this wave's */

    __device__ __forceinline__ void fetch(uint32_t now, uint32_t slot) const {
        Range(index + kDepth * now, index ? 4u * (uint64_t)(rows - kDepth * now) : 0u)
            .load<4>(at, held + SLOT * slot);
    }
};

template <class C>
struct TileRun {
    /* Load q of stage s is from at[q], in p or q moved on by s strides (both an operand's whole
     * extent from there). Operands of rows: of z, which lies inside them, those below Z;
     * p_z and q_z are an even q's, ^ 32 an odd one's. */
    const uint8_t *p_base, *q_base;
    uint64_t p_bytes, q_bytes, p_stride, q_stride;
    uint32_t p_at[C::DA], q_at[C::DB], p_z, q_z, Z;
    /* weight gradient: at[q] is z's row times the row's bytes and the column's place */
    Picks p_picks, q_picks;
    uint32_t p_row_bytes, q_row_bytes, p_col[C::DA], q_col[C::DB], q_late[2]; /* q_late: q_at[2, 3] next */
    uint32_t stages, wave, lane, wn, wt;

    __device__ __forceinline__ TileRun() {
        lane = threadIdx.x & 63u;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        wn = wave % C::WN, wt = wave / C::WN;
    }

    /* z of load q among the wave's eight */
    __device__ __forceinline__ uint32_t p_pick(int q) const { return 512u / C::BP * q + (lane >> 5); }
    __device__ __forceinline__ uint32_t q_pick(int q) const { return 4u * (q & 1) + (lane >> 4); }
    __device__ __forceinline__ void fetch_picks(uint32_t s) const {
        const uint32_t now = min(s, stages - 1u), slot = s % Picks::kRing;
        p_picks.fetch(now, slot);
        q_picks.fetch(now, slot);
    }
    __device__ __forceinline__ void read_picks(uint32_t s, uint32_t (&p)[C::DA], uint32_t (&q)[2]) const {
        const uint32_t slot = Picks::SLOT * (s % Picks::kRing);
        const uint32_t p_from = lds_addr(p_picks.held) + slot + 4u * p_pick(0);
        const uint32_t q_from = lds_addr(q_picks.held) + slot + 4u * q_pick(0);
        static_for<C::DA>([&](auto Q) { p[decltype(Q)::value] = ds_read4<8 * decltype(Q)::value>(p_from); });
        q[0] = ds_read4<0>(q_from), q[1] = ds_read4<16>(q_from);
    }
    /* A picked row's place: rows past the last, of the stage or of the tensor, lie past its end. The
     * products are of 24 bits: a row of up to 65535, its bytes. */
    __device__ __forceinline__ uint32_t place(const Picks &k, uint32_t read, uint32_t s, uint32_t z,
                                              uint32_t row_bytes, uint32_t col) const {
        const bool live = kDepth * min(s, stages - 1u) + z < k.rows;
        const uint32_t r = k.index ? live ? min(read, kMostPicked) : kMostPicked : z;
        return __umul24(r, row_bytes) + col;
    }
    __device__ __forceinline__ void set_picks(uint32_t s, uint32_t (&p)[C::DA], uint32_t (&q)[2]) {
        if constexpr (C::DIR != kWeight) return;
        else {
        static_for<C::DA>([&](auto I) {
            constexpr int i = decltype(I)::value;
            after_wait(p[i]);
            p_at[i] = place(p_picks, p[i], s, 8u * wave + p_pick(i), p_row_bytes, p_col[i]);
        });
        static_for<2>([&](auto I) {
            constexpr int i = decltype(I)::value;
            after_wait(q[i]);
            const uint32_t row = place(q_picks, q[i], s, 8u * wave + q_pick(i), q_row_bytes, 0u);
            q_at[i] = row + q_col[i];
            q_late[i] = row + q_col[2 + i];
        });
        }
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
            const Range r(q_base + q_stride * now, C::QCOLS ? q_bytes - q_stride * now : q_bytes);
            const bool in = C::QCOLS || kDepth * now + (q_z ^ 32u * (C::DB > 1 ? q & 1 : 0)) < Z;
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
        uint32_t p_lo, p_hi = 0u, q_lo, q_hi = 0u;
        if constexpr (C::PCOLS)
            p_lo = base + (col_slot<C::BP>(lane) ^ 128u * wn);
        else
            p_lo = base + 8192u * wn + lo, p_hi = base + 8192u * wn + hi;
        if constexpr (C::QCOLS)
            q_lo = base + C::A + (col_slot<128u>(lane) ^ 32u * wt);
        else
            q_lo = base + C::A + 2048u * wt + lo, q_hi = base + C::A + 2048u * wt + hi;
        Fragment<C::PCOLS> pf[4];
        Fragment<C::QCOLS> qf[2];
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
            if constexpr (C::QCOLS) {
                const uint32_t a = (q_lo + st) ^ (64u * (j & 3));
                static_for<2>([&](auto H) {
                    constexpr int h = decltype(H)::value, panel = 16384 * (j >> 2);
                    qf[j & 1].v[h][0] = ds_read_tr<panel + 128 * 64 * h>(a);
                    qf[j & 1].v[h][1] = ds_read_tr<panel + 128 * (64 * h + 8)>(a);
                });
            } else {
                qf[j & 1].v[0] = ds_read16<4096 * j>(q_lo + st);
                qf[j & 1].v[1] = ds_read16<4096 * j>(q_hi + st);
            }
        };
        auto barrier = [] {
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        };
        constexpr bool picks = C::DIR == kWeight;
        static_assert(!picks || C::EARLY, "rows are held for two stages on");
        uint32_t p_next[C::DA], q_next[2];
        auto rows_of_stage = [&](uint32_t s) {
            read_picks(s, p_next, q_next);
            wait_lgkm<0>();
            set_picks(s, p_next, q_next);
        };
        if constexpr (picks) {
#pragma unroll
            for (uint32_t s = 0; s < 3u; s++) fetch_picks(s);
            wait_vm<0>();
            rows_of_stage(0u);
            q_at[2] = q_late[0], q_at[3] = q_late[1];
        }
#pragma unroll
        for (int s = 0; s < C::STAGES - 1; s++) fetch<0, C::D>(smem, (uint32_t)s, (uint32_t)s);
        if constexpr (picks) {
            rows_of_stage(1u);
            q_at[2] = q_late[0], q_at[3] = q_late[1];
        }
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
            if constexpr (picks) { /* stage s + 2's have landed, s + 3's are loaded ahead of the rest */
                read_picks(s + 2u, p_next, q_next);
                fetch_picks(s + 3u);
            }
            if constexpr (TL == 1) fetch<0, C::D>(smem, ahead, to);
            next = slot;
            slot = slot + 1u == (uint32_t)C::STAGES ? 0u : slot + 1u;
            static_for<TL>([&](auto J) {
                constexpr int j = decltype(J)::value;
                constexpr bool last = j + 1 == TL;
                if constexpr (!last) read_q(std::integral_constant<int, j + 1>{});
                wait_lgkm<last ? 0 : C::QREADS>(); /* the next subtile's reads stay out */
                if constexpr (j == 0) static_for<4>([&](auto I) { pf[decltype(I)::value].ready(); });
                qf[j & 1].ready();
                if constexpr (picks && j == 0) set_picks(s + 2u, p_next, q_next);
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
            if constexpr (picks) q_at[2] = q_late[0], q_at[3] = q_late[1];
        }
        wait_lgkm<0>(); /* the reads past the end: their registers stay taken till here */
        static_for<4>([&](auto I) { pf[decltype(I)::value].ready(); });
        qf[0].ready();
        wait_vm<0>(); /* the loads past the end land before the LDS is used again */
    }
};

template <class C, uint32_t LDS>
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
    R.q_stride = 2u * kDepth;
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
    run_steps<C, LDS>(R, acc, smem, t.rows);
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
    for (uint32_t r = threadIdx.x / PIECES; r < t.rows; r += C::THREADS / PIECES) {
        const uint32_t to = rows[r];
        if (to != ~0u)
            *(uint4 *)((uint16_t *)A.out + (uint64_t)to * A.P + p0 + 8u * p) =
                *(const uint4 *)(smem + 16u * (PIECES * r + (p ^ (r & (PIECES - 1u)))));
    }
}

template <int DIR> using Tile32 = Tile<DIR, 4, 1, 4>;
template <int DIR> using Tile64 = Tile<DIR, 4, 2, 3>;
template <int DIR> using Tile128 = Tile<DIR, 4, 4, 3>;
template <int DIR> using Tile256 = Tile<DIR, 4, 8, 2>;

/* A block's class goes by the rows of its expert: a CU holds one block of any, so the
 * largest's registers and LDS cost the others nothing. */
template <int DIR>
__global__ __launch_bounds__(512, 2) void grouped_rows_kernel(GroupArgs A) {
    constexpr uint32_t LDS = Tile128<DIR>::LDS;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[LDS];
    RowTile t;
    uint32_t col;
    if (!find_tile(A, blockIdx.x, t, col) || t.rows == 0u) return;
    if (t.n <= 32u) row_tile<Tile32<DIR>, LDS>(A, smem, t, col);
    else if (t.n <= 64u) row_tile<Tile64<DIR>, LDS>(A, smem, t, col);
    else if (t.n <= 128u) row_tile<Tile128<DIR>, LDS>(A, smem, t, col);
    else row_tile<Tile256<DIR>, LDS>(A, smem, t, col);
}

/* 256 x 256 of an expert's weight gradient: p its columns (x), q its rows (dy). */
template <bool F32>
__global__ __launch_bounds__(512, 2) void grouped_weight_kernel(GroupArgs A) {
    using C = Tile<kWeight, 4, 8, 2>;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[C::LDS];
    const uint32_t works = A.E * A.tiles_p * A.tiles_q, each = (works + 7u) / 8u;
    uint32_t w = (blockIdx.x & 7u) * each + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= each || w >= works) return;
    const uint32_t expert = w / (A.tiles_p * A.tiles_q);
    w %= A.tiles_p * A.tiles_q;
    /* four q tiles at a time, along p */
    const uint32_t grp = w / (4u * A.tiles_p), in = w % (4u * A.tiles_p);
    const uint32_t high = min(4u, A.tiles_q - 4u * grp);
    const uint32_t p0 = C::BP * (in / high), q0 = C::BQ * (4u * grp + in % high);
    __shared__ uint8_t held[2][8][Picks::BYTES];
    TileRun<C> R;
    const uint32_t L = R.lane, at = L < 8u ? 4u * (8u * R.wave + L) : kNowhere;
    uint32_t row;
    const uint32_t rows = rows_of(A.offsets, expert, A.R, row);
    R.stages = (rows + kDepth - 1u) / kDepth;
    R.p_row_bytes = 2u * A.P, R.q_row_bytes = 2u * A.Q;
    R.p_picks = Picks{A.p_index ? A.p_index + row : nullptr, rows, at, held[0][R.wave]};
    R.q_picks = Picks{A.q_index ? A.q_index + row : nullptr, rows, at, held[1][R.wave]};
    /* picked rows lie anywhere in the tensor, others move on with the stages */
    R.p_stride = A.p_index ? 0u : (uint64_t)kDepth * R.p_row_bytes;
    R.q_stride = A.q_index ? 0u : (uint64_t)kDepth * R.q_row_bytes;
    R.p_base = (const uint8_t *)(A.p + (A.p_index ? 0u : (uint64_t)row * A.P) + p0);
    R.q_base = (const uint8_t *)(A.q + (A.q_index ? 0u : (uint64_t)row * A.Q) + q0);
    R.p_bytes = (uint64_t)(A.p_index ? A.p_rows : rows) * R.p_row_bytes - 2u * p0;
    R.q_bytes = (uint64_t)(A.q_index ? A.q_rows : rows) * R.q_row_bytes - 2u * q0;
#pragma unroll
    for (int q = 0; q < 4; q++) {
        R.p_col[q] = 2u * min(8u * col_dma_piece<C::BP>(L, C::DA * R.wave + (uint32_t)q), A.P - 8u - p0);
        const uint32_t ch = C::b_chunk(R.wave, (uint32_t)q);
        R.q_col[q] = 2u * min(128u * (ch >> 4) + 8u * col_dma_piece<128u>(L, ch & 15u), A.Q - 8u - q0);
    }
    const uint32_t high_q = min(C::BQ, A.Q - q0), width = min(C::BP, A.P - p0);
    f32x4 acc[C::TI][4];
    run_steps<C, C::LDS>(R, acc, smem, high_q);
    const uint32_t g = L >> 4, c = L & 15u;
    const uint64_t to = ((uint64_t)expert * A.Q + q0) * A.P + p0;
    if constexpr (F32) {
        if (A.accumulate && R.stages == 0u) return;
        float *out = (float *)A.out + to;
        static_for<C::TI>([&](auto J) {
            constexpr int j = decltype(J)::value;
            const uint32_t r = 16u * (2u * j + R.wt) + c;
            if (r >= high_q) return;
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++) {
                const uint32_t p = 64u * R.wn + 16u * i + 4u * g;
                if (p >= width) continue;
                f32x4 *place = (f32x4 *)(out + (uint64_t)r * A.P + p);
                f32x4 v = acc[j][i];
                if (A.accumulate) {
                    const f32x4 before = *place;
#pragma unroll
                    for (int k = 0; k < 4; k++) v[k] = __fadd_rn(before[k], v[k]);
                }
                *place = v;
            }
        });
    } else {
        uint16_t *out = (uint16_t *)A.out + to;
        constexpr uint32_t PIECES = C::BP / 8u;
        __syncthreads();
        static_for<C::TI>([&](auto J) {
            constexpr int j = decltype(J)::value;
            if (32u * j >= high_q) return;
            const uint32_t r = 16u * (2u * j + R.wt) + c;
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++) {
                const uint32_t p = 8u * R.wn + 2u * i + (g >> 1);
                *(uint2 *)(smem + 16u * (PIECES * r + (p ^ (r & (PIECES - 1u)))) + 8u * (g & 1u)) =
                    bf16x4(acc[j][i]);
            }
        });
        __syncthreads();
        const uint32_t p = threadIdx.x % PIECES;
        if (8u * p >= width) return;
        for (uint32_t r = threadIdx.x / PIECES; r < high_q; r += C::THREADS / PIECES)
            *(uint4 *)(out + (uint64_t)r * A.P + 8u * p) =
                *(const uint4 *)(smem + 16u * (PIECES * r + (p ^ (r & (PIECES - 1u)))));
    }
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
        overlap(output, out, weights, 2u * (uint64_t)experts * N * K))
        return false;
    GroupArgs A{};
    A.p = (const uint16_t *)weights, A.q = (const uint16_t *)input, A.offsets = offsets;
    A.q_index = input_index, A.to = output_index, A.q_rows = input_rows, A.to_rows = output_rows;
    A.out = output, A.R = rows, A.E = experts, A.P = P, A.Z = Z;
    A.tiles_p = (P + 255u) / 256u;
    /* n rows are in at most 1 + n / 256 tiles, of experts that have rows */
    const uint64_t tiles = rows / 256u + (experts < rows ? experts : rows);
    const uint64_t blocks = tiles * A.tiles_p + 8u;
    if (blocks >= 1u << 23) return false; /* 2^32 threads */
    hipLaunchKernelGGL(grouped_rows_kernel<DIR>, dim3((uint32_t)blocks), dim3(512), 0, st, A);
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
        overlap(output, out, input, 2u * (uint64_t)input_rows * columns))
        return false;
    GroupArgs A{};
    A.p = (const uint16_t *)input, A.q = (const uint16_t *)output_gradient, A.offsets = offsets;
    A.p_index = input_index, A.q_index = gradient_index, A.p_rows = input_rows, A.q_rows = gradient_rows;
    A.out = output, A.R = rows, A.E = expert_count, A.P = columns, A.Q = out_columns;
    A.accumulate = accumulate;
    A.tiles_p = (columns + 255u) / 256u, A.tiles_q = (out_columns + 255u) / 256u;
    const uint64_t blocks = 8u * (((uint64_t)expert_count * A.tiles_p * A.tiles_q + 7u) / 8u);
    if (blocks >= 1u << 23) return false;
    const auto kernel = f32 ? grouped_weight_kernel<true> : grouped_weight_kernel<false>;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)blocks), dim3(512), 0, (hipStream_t)stream, A);
    return hipGetLastError() == hipSuccess;
}
