// pdecode.cuh - attention of a few query rows per kv head over a paged cache: decode
// steps and short drafts, in groups of up to 16 rows (new tokens x query heads of a kv head).
//
// Bound: HBM; every key and value byte is read once and used for all rows at once.  The
// positions, not the rows, fill the 128 rows of the tensor cores' tile:
//   S^T [128 positions x rows] = K Q^T     A: the key tile as it lies in the pages
//   O^T [head_dim x rows]     += V^T P^T   A: the value tile, read along positions
// so a tile of 128 positions costs 16 products (bf16; 8 for e4m3) of about 70-90 cycles whatever the number of rows,
// against the ~2,800 (1,400) cycles that its bytes take at an SM's share of the measured
// HBM rate, and one thread per position has all rows' scores: its maximum over the
// positions is needed only when a score passes the running one, which one barrier with
// an "or" finds out.  A first version on warp-level matrix instructions with the rows as
// M = 16 spent 437 instructions per 16 positions and head, and took 228 us where this takes 102
// (32 sequences of 1,001 to 16,098 positions, 32 heads over 8, e4m3 pages).
//
// e4m3 codes are multiplied as they are.  A row of queries, scaled by a power of two so that its largest value lies
// in [128, 256), is two e4m3 rows q1 = rn(q), q2 = rn(2^5 (q - q1)) (|q - q1| <= 8), which hold a bf16 value's eight bits down
// to 2^-7 (smaller values are off by 2^-15 at most, 2^-22 of the row's largest).  A weight, its value row's exponent e
// taken into it, 2^(x - m + e - T + 11), is three e5m2 rows of three significant bits each: off by at most 2^-9 of itself, down
// to 2^-16.  T is a query row's own, the largest x - m + e that it sees (and up to 2^4 below later ones), so what the terms
// leave out is 2^-28 of the largest weighted value row that the query sees: neither a large row of little weight nor one that
// is hidden from it costs bits.  While the exponents of a run lie within 2^6, as those of most caches do, T is the largest
// exponent for all rows (2^-22); else it is found in a second look at the tile, in which rows of zeros do not count,
// whatever their exponent.
//
// Work split: the batch's positions are cut into blocks of 128 for each (sequence, kv head, group of
// 16 rows), a "pair" below, and the blocks, laid end to end, dealt evenly to the CTAs, whatever the
// lengths; a pair spread over several CTAs is joined by the last of them
// to finish, in order, so a call's bits do not depend on timing.
//
// Warps: 0-3 softmax, one thread per position of a tile and then per output dimension; 4
// issues the products (scores of the next tile before this tile's outputs); 5 loads by TMA, page by
// page, through a ring of tiles.  Every wait is bounded.
#pragma once

#include "pfill.cuh"

namespace oomb {

constexpr int kDecSoft = 128;               // softmax threads
constexpr int kDecThreads = kDecSoft + 64;
constexpr int kDecBlock = 128;              // positions of a work block: one tile
constexpr int kDecRows = 16;
constexpr int kDecCtas = 2;                 // CTAs of an SM
// Rows up to which a call comes here rather than to the 128-row tiles of prefill: two groups always, four while the pairs
// are no more than the SMs.  Over pages of 8 kv heads, here and there, in us: 32 rows 19 / 21 (one sequence of 2,000
// positions), 29 / 36 (one of 16,000), 38 / 50 (eight of 4,000) in bf16, 21 / 28, 29 / 43, 39 / 68 in e4m3; 64 rows 19 / 22,
// 34 / 37, 63 / 52 and 20 / 29, 36 / 43, 73 / 70; 128 rows 20 / 23, 51 / 38, 116 / 56.
constexpr int kDecRowsAlways = 32, kDecRowsFew = 64;

// Parts of a pair that one trip to L2 joins, and the blocks of a run that make more of them worth it: one sequence of 4,096
// bf16 positions over 8 kv heads takes 14.2 us in 8 parts, 11.8 in 16, 12.4 in 32; one of 16,000 takes 20.1 us in the 16
// that runs of 8 blocks make, 20.6 in 21 and 22.3 in 31; one of 60,000 48 us in the 37 that fill the SMs.
constexpr int kDecParts = 16, kDecRun = 8;

// e4m3.  Weights are made as 2^(x - n + 11 - 30) 2^(e - X + 30), X the largest exponent byte met and n = m - (X - T): the left
// factor is what the sum of weights adds up, and stays an fp32 number (2^97 a position) while exponents lie within 2^112.  (n
// is only a reference: what it loses where m is large cancels, but past 2^20 it could no longer hold X - T.)
// Over 8 kv heads, eight sequences of 4,000 positions and 16 rows take 29.2 us if every run looks twice, 26.8 if only those past
// 2^6 do; one of 4,096 and 4 rows 12.6 and 11.4.
constexpr int kDecUnit = 30, kDecSpread = 112, kDecNear = 6;
constexpr float kRestUp = 32.0f;  // what q - q1 is multiplied by
constexpr int kZeroByte = 127;  // the exponent that an append gives a row of zeros

enum : unsigned {
    ERR_DEC_WAIT = 0xb00,  // a decode pipeline wait ran out (+ the waiting role)
};

// R: rows a tile is made for (4, 8 or 16; a call's rows at most).
template <int KIND, int D, int R>
struct DecodeGeo {
    static constexpr bool F8 = KIND == KV_E4M3;
    static constexpr int ROW = F8 ? D : 2 * D;                  // bytes of a position's row
    static constexpr int CHUNK = ROW < 128 ? ROW : 128;         // bytes of a swizzled row
    static constexpr int CH = ROW / CHUNK;
    static constexpr int TILE = kDecBlock * ROW;
    // terms of a query and of a weight: a product takes 16 columns whatever their number, so bf16 weights of up to 8 rows are two
    // bf16 terms (off by 2^-15) for nothing; with 16 rows the second would take the third tile's room, and they are one (2^-8)
    static constexpr int QT = F8 ? 2 : 1, PT = F8 ? 3 : R <= 8 ? 2 : 1;
    static constexpr int NQ = (R * QT + 15) / 16 * 16, NP = (R * PT + 15) / 16 * 16;
    static constexpr int Q_BYTES = (CH * NQ * CHUNK + 1023) / 1024 * 1024;
    static constexpr int P_STEP = (NP * kDecBlock * (F8 ? 1 : 2) + 1023) / 1024 * 1024;
    static constexpr int EXPS = 8;                              // tiles whose exponents are kept
    static constexpr int BARS = 1408;                           // bytes of the barriers and of what the warps tell one another
    static constexpr int REST = Q_BYTES + 2 * P_STEP + (F8 ? EXPS * 2 * kDecBlock : 0) + BARS;
    static constexpr int ROOM = 228 * 1024 / kDecCtas - 1024 - REST;
    static constexpr int STAGES = ROOM / TILE < 8 ? ROOM / TILE : 8;
    static constexpr int Q_OFF = STAGES * TILE;
    static constexpr int P_OFF = Q_OFF + Q_BYTES;
    static constexpr int EXP_OFF = P_OFF + 2 * P_STEP;
    static constexpr int BAR_OFF = EXP_OFF + (F8 ? EXPS * 2 * kDecBlock : 0);
    static constexpr int TOTAL = BAR_OFF + BARS;
    static constexpr int S_COLS = 32;                           // tensor-memory columns of a score buffer
    static constexpr int PAD = D + 4;                           // floats of a partial row
    static_assert(NQ <= S_COLS && NP <= 64, "tensor memory");
    static_assert(kDecCtas * (TOTAL + 1024) <= 228 * 1024, "shared memory");
};

struct DecodeWs {
    unsigned* counters;  // [grid] arrivals, zero between launches
    float* part;         // [2 * grid][rows][D + 4]: acc, m, l
    int rows;
};

struct DecodeBars {
    uint64_t kv_full[8], kv_empty[8], s_full[2], p_ready[2], p_free[2], q_ready, e_full[8], done;
    uint32_t tmem;
    unsigned beat;  // moves while rows are done again
    float red[4][kDecRows], redt[4][kDecRows];
    float scale[kDecRows];    // e4m3: a row's scale, its power of two in it
    float n[kDecRows], top[kDecRows], T[kDecRows], fl[kDecRows], fo[kDecRows];  // a row's reference, largest score, T, and factors of a change
    int redx[4], redn[4], redv[4];
    unsigned last;
    int4 start;               // the CTA's first sequence, its first block, the blocks of its pairs, its groups
    Seq start_seq;
    int2 sum[kDecThreads / 32];
};

// W blocks dealt to S CTAs in proportion: CTA c begins at W c / S, so that with as many CTAs for each of equally long pairs
// none has parts of two.  In 32 bits wherever W S fits: a 64-bit division takes some 200 ns here.
struct DecodeDeal {
    unsigned W, S;
    __device__ bool narrow() const { return __umulhi(W, S) == 0; }
    __device__ int lo(int c) const {
        return narrow() ? static_cast<int>(W * static_cast<unsigned>(c) / S) : static_cast<int>(static_cast<unsigned long long>(W) * c / S);
    }
    // the last CTA that begins at or before the block
    __device__ int owner(int block) const {
        return narrow() ? static_cast<int>(((block + 1u) * S - 1u) / W) : static_cast<int>(((block + 1ull) * S - 1) / W);
    }
};

// Descriptors' high words: 128-byte rows in the 128-byte swizzle (8-row groups 1024 bytes apart), or 64-byte rows in the
// 64-byte one (512).
__host__ __device__ constexpr uint32_t dec_desc_hi(int chunk) {
    return chunk == 128 ? (64u | (1u << 14) | (2u << 29)) : (32u | (1u << 14) | (4u << 29));
}
// Byte of 16-byte chunk c of row r in such a layout.
__device__ __forceinline__ int dec_swizzle(int chunk, int r, int c) {
    return chunk == 128 ? r * 128 + ((c ^ (r & 7)) << 4) : r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
}

template <bool F8>
__device__ __forceinline__ void dec_mma(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t a_hi, uint32_t b_hi, uint32_t idesc, int acc) {
    if constexpr (F8)
        asm volatile(
            "{\n .reg .pred p;\n .reg .b64 da, db;\n setp.ne.b32 p, %6, 0;\n mov.b64 da, {%1, %3};\n mov.b64 db, {%2, %4};\n"
            " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %5, p;\n}" ::"r"(d),
            "r"(a_lo), "r"(b_lo), "r"(a_hi), "r"(b_hi), "r"(idesc), "r"(acc)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred p;\n .reg .b64 da, db;\n setp.ne.b32 p, %6, 0;\n mov.b64 da, {%1, %3};\n mov.b64 db, {%2, %4};\n"
            " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n}" ::"r"(d),
            "r"(a_lo), "r"(b_lo), "r"(a_hi), "r"(b_hi), "r"(idesc), "r"(acc)
            : "memory");
}

template <int N>
__device__ __forceinline__ void tm_ld(uint32_t t, float* v) {
    static_assert(N % 16 == 0, "sixteen columns at a time");
#pragma unroll
    for (int c = 0; c < N; c += 16) tm_ld16(t + c, v + c);
    tc_wait_ld();
}

__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&h);
}
// (lo, hi) to two e5m2 codes (or e4m3), and what they leave of the two values.
__device__ __forceinline__ unsigned split_e5m2(float& lo, float& hi) {
    unsigned short c;
    unsigned h;
    asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(c) : "f"(hi), "f"(lo));
    asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(h) : "h"(c));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    lo -= f.x;
    hi -= f.y;
    return c;
}
__device__ __forceinline__ unsigned split_e4m3(float& lo, float& hi) {
    unsigned short c;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(c) : "f"(hi), "f"(lo));
    const float2 f = e4m3x2_to_float2(c);
    lo -= f.x;
    hi -= f.y;
    return c;
}

// A sequence's rows of a kv head go in groups of kDecRows, each with the blocks of its own: a "pair" below is one
// (sequence, kv head, group).
__device__ __forceinline__ int dec_groups(const Seq& s, int G) { return (s.n * G + kDecRows - 1) / kDecRows; }
__device__ __forceinline__ int dec_blocks(const Seq& s, int max_q) {
    return s.n == 0 || s.n > max_q ? 0 : max(1, (s.len + kDecBlock - 1) / kDecBlock);  // without positions, still its zeros
}

// A run of blocks of one pair.
struct DecodeSeg {
    Seq sq;
    int b, kvh, row0, rows, tok0, tok1, tiles;
    int pair_first, pair_end, lo;
};

// Walks a CTA's segments in order; every role does so on its own.
struct DecodeWalk {
    DecodeDeal deal;
    int lo, hi;      // this CTA's blocks yet to come
    int b, b_first;  // a sequence and its first block
    Seq sq;
    int nb, groups;  // its blocks of a pair, its groups
    __device__ bool next(const PattnParams& p, DecodeSeg& g) {
        if (lo >= hi) return false;
        while (lo >= b_first + nb * groups * p.Hkv) {
            b_first += nb * groups * p.Hkv;
            b++;
            sq = read_seq(p.q_start, p.kv_len, b, p.T, p.kv_max, nullptr);
            nb = dec_blocks(sq, p.max_q);
            groups = dec_groups(sq, p.G);
        }
        const int pair = (lo - b_first) / nb;
        g.sq = sq;
        g.b = b;
        g.kvh = pair / groups;
        g.row0 = (pair - g.kvh * groups) * kDecRows;
        g.rows = min(kDecRows, sq.n * p.G - g.row0);
        g.pair_first = b_first + pair * nb;
        g.pair_end = g.pair_first + nb;
        g.lo = lo;
        const int end = min(g.pair_end, hi);
        g.tok0 = (lo - g.pair_first) * kDecBlock;
        g.tok1 = min(sq.len, (end - g.pair_first) * kDecBlock);
        g.tiles = g.tok1 > g.tok0 ? (g.tok1 - g.tok0 + kDecBlock - 1) / kDecBlock : 0;
        lo = end;
        return true;
    }
};

template <int KIND, int D, int R>
__global__ void __launch_bounds__(kDecThreads, kDecCtas)
    decode_rows_kernel(const __grid_constant__ PattnParams p, const __grid_constant__ DecodeWs ws, const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap) {
    using Geo = DecodeGeo<KIND, D, R>;
    constexpr bool F8 = Geo::F8;
    constexpr int ST = Geo::STAGES, CHUNK = Geo::CHUNK, CH = Geo::CH, PAD = Geo::PAD;
    extern __shared__ __align__(1024) uint8_t smem[];
    DecodeBars* bar = reinterpret_cast<DecodeBars*>(smem + Geo::BAR_OFF);
    static_assert(sizeof(DecodeBars) <= Geo::BARS, "barriers");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (smem_addr(smem) & 1023u) {  // the swizzle's pattern starts there
        if (tid == 0) record_error(p.err, ERR_DEC_WAIT + 15);
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < ST; i++) {
            mbar_init(&bar->kv_full[i], 1);
            mbar_init(&bar->kv_empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&bar->s_full[i], 1);
            mbar_init(&bar->p_ready[i], 4);
            mbar_init(&bar->p_free[i], 1);
        }
        for (int i = 0; i < Geo::EXPS; i++) mbar_init(&bar->e_full[i], 1);
        mbar_init(&bar->q_ready, 4);
        mbar_init(&bar->done, 1);
        bar->beat = 0;
        fence_barrier_init();
    }
    if (warp == 4) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 128;" ::"r"(smem_addr(&bar->tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bar->tmem, o_col = tmem + 2 * Geo::S_COLS;
    pdl_wait();
    pdl_launch_dependents();

    // ---- this CTA's blocks of the batch ----
    DecodeWalk walk{};
    {
        Seq seen{};
        int pairs_of = 0;  // a sequence's pairs
        auto blocks_of = [&](int b) {
            pairs_of = 0;
            if (b >= p.B) return 0;
            seen = read_seq(p.q_start, p.kv_len, b, p.T, p.kv_max, p.err);
            if (seen.n > p.max_q) record_error(p.err, ERR_KV_SEQ);
            pairs_of = dec_groups(seen, p.G) * p.Hkv;
            return dec_blocks(seen, p.max_q) * pairs_of;
        };
        int total = 0, pairs = 0, mine = 0;
        for (int b0 = 0; b0 < p.B; b0 += kDecThreads) {
            mine = blocks_of(b0 + tid);
            const int v = __reduce_add_sync(0xffffffffu, mine), n = __reduce_add_sync(0xffffffffu, mine > 0 ? pairs_of : 0);
            if (lane == 0) bar->sum[warp] = make_int2(v, n);
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kDecThreads / 32; w++) {
                total += bar->sum[w].x;
                pairs += bar->sum[w].y;
            }
            __syncthreads();
        }
        // As many CTAs as blocks, or as are resident.  Few pairs: equally many CTAs each, at least kDecParts, and more only for
        // kDecRun blocks a CTA or more (the end and the beginning of a run cost as much as three or four blocks, and a
        // launch that leaves room lets the next begin beside it).
        const int W = total, grid = gridDim.x;  // fits: checked by the caller for the longest sequences
        int S = min(W, grid);
        if (pairs > 0 && 2 * pairs <= grid)
            S = min(S, pairs * min(grid / pairs, max(kDecParts, W / (pairs * kDecRun))));
        if (static_cast<int>(blockIdx.x) < S) {
            walk.deal.W = W;
            walk.deal.S = S;
            walk.lo = walk.deal.lo(blockIdx.x);
            walk.hi = walk.deal.lo(blockIdx.x + 1);
            int prefix = 0;
            for (int b0 = 0; b0 < p.B; b0 += kDecThreads) {
                if (p.B > kDecThreads) mine = blocks_of(b0 + tid);
                int inc = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int u = __shfl_up_sync(0xffffffffu, inc, o);
                    if (lane >= o) inc += u;
                }
                if (lane == 31) bar->sum[warp].x = inc;
                __syncthreads();
                int end = prefix + inc;
                for (int w = 0; w < warp; w++) end += bar->sum[w].x;
                if (mine > 0 && end - mine <= walk.lo && walk.lo < end) {
                    bar->start = make_int4(b0 + tid, end - mine, mine / pairs_of, pairs_of / p.Hkv);
                    bar->start_seq = seen;
                }
#pragma unroll
                for (int w = 0; w < kDecThreads / 32; w++) prefix += bar->sum[w].x;
                __syncthreads();
            }
            walk.b = bar->start.x;
            walk.b_first = bar->start.y;
            walk.nb = bar->start.z;
            walk.groups = bar->start.w;
            walk.sq = bar->start_seq;
        }
    }
    DecodeSeg g;
    if (warp == 5) {
        // ---- loader ----
        Ring<ST> r;
        bool ok = true;
        unsigned tile_no = 0;
        const int per_tile = kDecBlock >> p.kv.page_log2, page = 1 << p.kv.page_log2;
        while (ok && walk.next(p, g)) {
            if (g.tiles == 0) continue;
            const int32_t* table = p.kv.table + static_cast<int64_t>(g.b) * p.kv.table_stride;
            auto lookup = [&](int i) {
                const int at = (g.tok0 >> p.kv.page_log2) + i * per_tile + lane;
                return i < g.tiles && lane < per_tile && at < p.kv.max_pages ? __ldcg(table + at) : 0;
            };
            auto load = [&](bool value, int i, int id) {
                if (!ok || !fa_wait(&bar->kv_empty[r.i], r.phase ^ 1, p.err, ERR_DEC_WAIT + 1, &bar->beat)) {
                    ok = false;
                    return;
                }
                uint8_t* dst = smem + r.i * Geo::TILE;
                uint64_t* full = &bar->kv_full[r.i];
                const int have = min(per_tile, (g.tok1 - g.tok0 - i * kDecBlock + page - 1) >> p.kv.page_log2);
                const bool mine = lane < have, good = mine && id >= 0 && id < p.kv.num_pages;
                if (mine && !good && !value) record_error(p.err, ERR_KV_TABLE);
                if (lane == 0) mbar_arrive_expect_tx(full, have * page * Geo::ROW);
                const unsigned e = tile_no & (Geo::EXPS - 1);
                uint8_t* exps = smem + Geo::EXP_OFF + e * 2 * kDecBlock;
                if (F8 && !value) {  // both kinds' exponents come with the keys
                    if (mine && !good)
                        for (int o = 0; o < page; o += 16) {
                            *reinterpret_cast<uint4*>(exps + lane * page + o) = make_uint4(0u, 0u, 0u, 0u);
                            *reinterpret_cast<uint4*>(exps + kDecBlock + lane * page + o) = make_uint4(0u, 0u, 0u, 0u);
                        }
                    const int n = __popc(__ballot_sync(0xffffffffu, good));
                    if (lane == 0) mbar_arrive_expect_tx(&bar->e_full[e], n * page * 2);
                }
                __syncwarp();
                if (mine) {
                    const int at = good ? id : p.kv.num_pages;  // outside the map: zeros
#pragma unroll
                    for (int c = 0; c < CH; c++)
                        tma_load_4d(dst + c * kDecBlock * CHUNK + lane * page * CHUNK, value ? &vmap : &kmap, c * 64, 0, g.kvh, at, full);
                    if (F8 && !value && good) {
                        const int64_t from = id * p.kv.exp_stride + (static_cast<int64_t>(g.kvh) << p.kv.page_log2);
                        bulk_g2s_plain(exps + lane * page, p.kv.ke + from, page, &bar->e_full[e]);
                        bulk_g2s_plain(exps + kDecBlock + lane * page, p.kv.ve + from, page, &bar->e_full[e]);
                    }
                }
                if (!value) tile_no++;
                r.next();
            };
            int cur = lookup(0), nxt = lookup(1);
            load(false, 0, cur);
            for (int i = 0; i < g.tiles && ok; i++) {
                const int was = cur;
                if (i + 1 < g.tiles) {
                    cur = nxt;
                    nxt = lookup(i + 2);
                    load(false, i + 1, cur);
                }
                load(true, i, was);
            }
        }
        // the last loads of every slot have landed before the CTA ends, whoever still waited for them: nothing may arrive in its
        // shared memory later (a slot never loaded counts as landed)
        for (int i = 0; i < ST; i++) {
            fa_drain(&bar->kv_full[r.i], r.phase ^ 1, p.err, ERR_DEC_WAIT + 2);
            r.next();
        }
        for (unsigned e = 0; F8 && e < Geo::EXPS && e < tile_no; e++)
            fa_drain(&bar->e_full[e], ((tile_no - 1 - e) / Geo::EXPS) & 1, p.err, ERR_DEC_WAIT + 2);
    } else if (warp == 4) {
        // ---- the issuing warp ----
        Ring<ST> r;
        unsigned t = 0, q_ph = 0;  // tiles so far
        bool ok = true;
        bool gone = false;  // this lane gave up
        auto wait = [&](uint64_t* b, unsigned ph, int role) { gone |= !fa_wait_lane(b, ph, p.err, ERR_DEC_WAIT + role, &bar->beat); };
        constexpr uint32_t fmt = F8 ? 0u : (1u << 7) | (1u << 10);
        constexpr uint32_t id_s = (1u << 4) | fmt | (static_cast<uint32_t>(Geo::NQ >> 3) << 17) | (8u << 24);
        // A along positions (bit 15); e4m3 values with e5m2 weights
        constexpr uint32_t id_o = (1u << 4) | fmt | (F8 ? 1u << 10 : 0u) | (1u << 15) | (static_cast<uint32_t>(Geo::NP >> 3) << 17) | (8u << 24);
        constexpr uint32_t hi = dec_desc_hi(CHUNK), p_hi = dec_desc_hi(128);
        // the next 64-column chunk of a bf16 value tile; with one chunk of 64 dimensions the rows above repeat it, unread
        constexpr uint32_t lead = D == 128 && !F8 ? (kDecBlock * CHUNK) >> 4 : 0;
        const uint32_t base = uniform(smem_addr(smem) >> 4), tm = uniform(tmem), oc = uniform(o_col);
        auto scores = [&](int stage, unsigned tile) {
            tc_fence_after();
            const uint32_t a = uniform((base + stage * (Geo::TILE >> 4)) | (1u << 16)), q = (base + (Geo::Q_OFF >> 4)) | (1u << 16);
            const uint32_t d = uniform(tm + (tile & 1) * Geo::S_COLS);
            uint64_t* const done = &bar->s_full[tile & 1];
            if (elect_one()) {
#pragma unroll
                for (int i = 0; i < Geo::ROW / 32; i++) {
                    const uint32_t ao = ((i * 32 / CHUNK) * kDecBlock * CHUNK + i * 32 % CHUNK) >> 4;
                    const uint32_t bo = ((i * 32 / CHUNK) * Geo::NQ * CHUNK + i * 32 % CHUNK) >> 4;
                    dec_mma<F8>(d, a + ao, q + bo, hi, hi, id_s, i > 0);
                }
                tc_commit(done);
            }
            __syncwarp();
        };
        auto outputs = [&](int stage, unsigned tile, bool first) {
            tc_fence_after();
            const uint32_t a = uniform((base + stage * (Geo::TILE >> 4)) | (lead << 16));
            const uint32_t w = uniform((base + (Geo::P_OFF >> 4) + (tile & 1) * (Geo::P_STEP >> 4)) | (1u << 16));
            const int more = uniform(!first);
            uint64_t* const done = &bar->p_free[tile & 1];
            if (elect_one()) {
                constexpr int K = F8 ? 32 : 16;  // positions of a product
#pragma unroll
                for (int i = 0; i < kDecBlock / K; i++) {
                    const uint32_t bo = F8 ? (i * 32) >> 4 : ((i / 4) * Geo::NP * 128 + (i % 4) * 32) >> 4;
                    dec_mma<F8>(oc, a + ((i * K * CHUNK) >> 4), w + bo, hi, p_hi, id_o, i > 0 ? 1 : more);
                }
                tc_commit(done);
            }
            __syncwarp();
        };
        auto release = [&](int stage) {
            if (elect_one()) tc_commit(&bar->kv_empty[stage]);
            __syncwarp();
        };
        while (ok && walk.next(p, g)) {
            if (g.tiles == 0) continue;
            wait(&bar->q_ready, q_ph, 3);
            q_ph ^= 1;
            wait(&bar->kv_full[r.i], r.phase, 4);
            scores(r.i, t);
            release(r.i);
            r.next();
            for (int i = 0; i < g.tiles && ok; i++, t++) {
                if (i + 1 < g.tiles) {
                    wait(&bar->kv_full[r.i], r.phase, 4);
                    scores(r.i, t + 1);
                    release(r.i);
                    r.next();
                }
                wait(&bar->kv_full[r.i], r.phase, 4);
                const int left = g.tok1 - g.tok0 - i * kDecBlock;
                if (left < kDecBlock) {
                    // rows behind the last position: anything may be there, and 0 * NaN is NaN
                    uint8_t* v = smem + r.i * Geo::TILE;
                    for (int o = left * (CHUNK / 16) + lane; o < kDecBlock * (CHUNK / 16); o += 32)
#pragma unroll
                        for (int c = 0; c < CH; c++) *reinterpret_cast<uint4*>(v + c * kDecBlock * CHUNK + o * 16) = make_uint4(0u, 0u, 0u, 0u);
                    fence_async_smem();
                    __syncwarp();
                }
                wait(&bar->p_ready[t & 1], (t >> 1) & 1, 5);
                outputs(r.i, t, i == 0);
                release(r.i);
                r.next();
                ok = !__any_sync(0xffffffffu, gone);
            }
        }
        // every product has read its operands before the CTA ends, also where the softmax gave up on one
        if (elect_one()) tc_commit(&bar->done);
        __syncwarp();
        fa_drain(&bar->done, 0, p.err, ERR_DEC_WAIT + 11);
    } else {
        // ---- softmax: a position's thread, then an output dimension's ----
        const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
        constexpr float kSlack = F8 ? 4.0f : 8.0f, kBase = F8 ? 11.0f - kDecUnit : -kFaDown;
        unsigned t = 0, v_item = 0;  // tiles so far, and what the loader brought before the segment
        bool stop = false;
        // the four warps meet; whether any says so
        auto meet = [&](bool any) {
            unsigned x;
            asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 q, %1, 0;\n bar.red.or.pred p, 1, 128, q;\n selp.u32 %0, 1, 0, p;\n}"
                         : "=r"(x)
                         : "r"(static_cast<unsigned>(any))
                         : "memory");
            return x != 0;
        };
        // A thread whose wait ran out goes on to the next meeting, where all learn of it: none leaves the others waiting there.
        bool gone = false;
        auto wait = [&](uint64_t* b, unsigned ph, int role) {
            if (!fa_wait_lane(b, ph, p.err, ERR_DEC_WAIT + role, &bar->beat)) gone = true;
        };
        while (!stop && walk.next(p, g)) {
            const Seq sq = g.sq;
            const int rows = g.rows, row0 = g.row0;
            float m[R], l[R], sc[R];  // sc: e4m3, up to 8 rows (16 read it from shared memory, 84 bytes of spills less)
            int vis[R];
#pragma unroll
            for (int r = 0; r < R; r++) {
                m[r] = -INFINITY;
                l[r] = 0.0f;
                vis[r] = r < rows ? max(0, min(sq.len, sq.len - sq.n + (row0 + r) / p.G + 1)) : 0;
            }
            int X = 0;       // e4m3: the exponent byte that the outputs are counted in
            int low = 255;   // the least of this thread's positions
            bool thin = false;  // one of them raised a reference with codes below 2
            bool wide = false;  // the exponents lie apart
            if (F8 && tid < R) bar->n[tid] = bar->top[tid] = -INFINITY;
            if (g.tiles > 0) {
                // ---- the queries as the scores' second operand; the last segment's scores are all made ----
                if constexpr (!F8) {
                    for (int o = tid; o < R * (D / 8); o += kDecSoft) {
                        const int r = o / (D / 8), c = o % (D / 8);
                        uint4 x = make_uint4(0u, 0u, 0u, 0u);
                        if (r < rows)
                            x = __ldcg(reinterpret_cast<const uint4*>(p.q + static_cast<int64_t>(sq.q0 + (row0 + r) / p.G) * p.q_stride +
                                                                      static_cast<int64_t>(g.kvh * p.G + (row0 + r) % p.G) * D + c * 8));
                        *reinterpret_cast<uint4*>(smem + Geo::Q_OFF + (c / 8) * Geo::NQ * 128 + dec_swizzle(128, r, c % 8)) = x;
                    }
                } else {
                    // a row by 8 threads, D / 8 values each
                    constexpr int V = D / 8;
                    for (int r0 = 0; r0 < R; r0 += kDecSoft / 8) {
                        const int r = r0 + tid / 8, c = tid % 8;
                        float f[V];
                        float big = 0.0f;
                        const bool in = r < rows;
                        const uint16_t* q = p.q + static_cast<int64_t>(sq.q0 + (in ? (row0 + r) / p.G : 0)) * p.q_stride +
                                            static_cast<int64_t>(g.kvh * p.G + (in ? (row0 + r) % p.G : 0)) * D + c * V;
#pragma unroll
                        for (int i = 0; i < V; i += 8) {
                            const uint4 x = in ? __ldcg(reinterpret_cast<const uint4*>(q + i)) : make_uint4(0u, 0u, 0u, 0u);
                            const unsigned u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                f[i + 2 * k] = __uint_as_float(u[k] << 16);
                                f[i + 2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
                                big = fmaxf(big, fmaxf(fabsf(f[i + 2 * k]), fabsf(f[i + 2 * k + 1])));
                            }
                        }
#pragma unroll
                        for (int o = 1; o < 8; o <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
                        const int ex = max(-126, static_cast<int>(__float_as_uint(big) >> 23) - 127 - 7);  // 2^ex and 2^-ex are fp32 numbers
                        const float up = power_of(-ex);
                        if (r < R) {
                            if (c == 0) bar->scale[r] = p.scale_log2 * power_of(ex);
                            // a value that is not finite has no code: its row's scores become NaN
                            const bool bad = !(big <= 3.4e38f);
                            uint8_t* q1 = smem + Geo::Q_OFF;
#pragma unroll
                            for (int i = 0; i < V; i += 4) {
                                float a = f[i] * up, b = f[i + 1] * up, d = f[i + 2] * up, e = f[i + 3] * up;
                                if (a != a || b != b || d != d || e != e || bad) a = __uint_as_float(0x7fffffffu);
                                const unsigned h0 = split_e4m3(a, b), h1 = split_e4m3(d, e);
                                a *= kRestUp, b *= kRestUp, d *= kRestUp, e *= kRestUp;
                                const unsigned l0 = split_e4m3(a, b), l1 = split_e4m3(d, e);
                                const int at = c * V + i;  // byte of the row
                                *reinterpret_cast<unsigned*>(q1 + dec_swizzle(CHUNK, r, at / 16) + at % 16) = h0 | (h1 << 16);
                                *reinterpret_cast<unsigned*>(q1 + dec_swizzle(CHUNK, R + r, at / 16) + at % 16) = l0 | (l1 << 16);
                            }
                        }
                    }
                }
                fence_async_smem();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar->q_ready);
                if constexpr (F8) {
                    meet(false);
#pragma unroll
                    for (int r = 0; r < R; r++) sc[r] = R <= 8 ? bar->scale[r] : 0.0f;
                }
            }
            for (int i = 0; i < g.tiles; i++, t++) {
                wait(&bar->s_full[t & 1], (t >> 1) & 1, 6);
                tc_fence_after();
                float s[Geo::NQ];
                tm_ld<Geo::NQ>(tmem + lanes + (t & 1) * Geo::S_COLS, s);
                const int tok = g.tok0 + i * kDecBlock + tid;
                int ve = 0;
                float kf = 1.0f;
                if constexpr (F8) {
                    const unsigned e = t & (Geo::EXPS - 1);
                    wait(&bar->e_full[e], (t / Geo::EXPS) & 1, 7);
                    const uint8_t* ep = smem + Geo::EXP_OFF + e * 2 * kDecBlock;
                    kf = exp_byte(ep[tid]);
                    if (tok < g.tok1) {
                        ve = ep[kDecBlock + tid];
                        if (ve) low = min(low, ve);  // 0: a bad table entry's zeros
                    }
                }
                // (2^(e - X + 30) is to stay an fp32 number)
                bool over = F8 && (ve > X + 60 || (!wide && low + kDecNear < X));
                const float top = kSlack + static_cast<float>(X - ve);
#pragma unroll
                for (int r = 0; r < R; r++) {
                    float x = F8 ? fmaf(s[R + r], 1.0f / kRestUp, s[r]) * ((R <= 8 ? sc[r] : bar->scale[r]) * kf) : s[r] * p.scale_log2;
                    if (tok >= vis[r]) x = -INFINITY;
                    s[r] = x;
                    over |= x > m[r] + top || (m[r] == -INFINITY && x != -INFINITY);
                }
                if (meet(over || gone)) {
                    // the tile's maxima over its positions, and the outputs so far brought to them
#pragma unroll
                    for (int r = 0; r < R; r++) {
                        float x;
                        asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(x) : "f"(s[r]));
                        if (lane == 0) bar->red[warp][r] = x;
                    }
                    if constexpr (F8) {
                        const int x = __reduce_max_sync(0xffffffffu, over ? ve : 0), n = __reduce_min_sync(0xffffffffu, low);
                        const bool none = __any_sync(0xffffffffu, over && ve == kZeroByte);
                        if (lane == 0) {
                            bar->redx[warp] = x;
                            bar->redn[warp] = none ? -1 : n;  // a row of zeros, maybe
                        }
                    }
                    if (i > 0) wait(&bar->p_free[(t - 1) & 1], ((t - 1) >> 1) & 1, 8);  // the outputs are at rest
                    if (meet(gone)) {
                        stop = true;
                        break;
                    }
                    float f[R];
                    auto over_warps = [&](const float (&x)[4][kDecRows], int r) { return fmaxf(fmaxf(x[0][r], x[1][r]), fmaxf(x[2][r], x[3][r])); };
                    if constexpr (F8) {
                        int xn = max(max(X, max(bar->redx[0], bar->redx[1])), max(bar->redx[2], bar->redx[3]));
                        const int ln = min(min(bar->redn[0], bar->redn[1]), min(bar->redn[2], bar->redn[3]));
                        const bool look = wide || ln < 0 || xn - ln > kDecNear;
                        if (look) {
                            // ---- the second look: how large this tile's weighted value rows are ----
                            if (__any_sync(0xffffffffu, over)) {  // what these positions' value rows hold
                                const unsigned item = v_item + (i + 1 < g.tiles ? 2 * i + 2 : 2 * g.tiles - 1);
                                wait(&bar->kv_full[item % ST], (item / ST) & 1, 10);
                                const uint8_t* row = smem + (item % ST) * Geo::TILE + tid * CHUNK;
                                unsigned bits = 0;
#pragma unroll
                                for (int c = 0; c < CHUNK / 16; c++) {
                                    const uint4 w = *reinterpret_cast<const uint4*>(row + (((c + tid) % (CHUNK / 16)) << 4));
                                    bits |= w.x | w.y | w.z | w.w;
                                }
                                if (over && (bits & 0x7f7f7f7fu) == 0) ve = 0;
                                thin |= over && ve > 0 && (bits & 0x40404040u) == 0;
                            }
                            const int v = __reduce_max_sync(0xffffffffu, over ? ve : 0);
                            if (lane == 0) bar->redv[warp] = v;
#pragma unroll
                            for (int r = 0; r < R; r++) {
                                float y = ve == 0 ? -INFINITY : (s[r] - over_warps(bar->red, r)) + static_cast<float>(ve);
                                asm volatile("redux.sync.max.f32 %0, %0, 0xffffffff;" : "+f"(y));
                                if (lane == 0) bar->redt[warp][r] = y;
                            }
                            if (meet(gone)) {
                                stop = true;
                                break;
                            }
                            xn = max(max(X, max(bar->redv[0], bar->redv[1])), max(bar->redv[2], bar->redv[3]));
                        }
                        if (tid < R) {  // a row's thread
                            const float was = bar->n[tid], tile = over_warps(bar->red, tid), mx = fmaxf(bar->top[tid], tile);
                            const bool first = was == -INFINITY;
                            float n = mx;
                            if (look) {
                                // (an X that stood for T may have come from rows of zeros: too low a T costs nothing, the outputs are fp32)
                                const float old = first ? -INFINITY : wide ? bar->T[tid] + (bar->top[tid] - mx) : (was - mx) + static_cast<float>(X) - 60.0f;
                                const float T = ceilf(fmaxf(over_warps(bar->redt, tid) + (tile - mx), old));
                                n = mx - (static_cast<float>(xn) - fmaxf(T, static_cast<float>(xn - kDecSpread)));
                                bar->T[tid] = T;
                            }
                            bar->n[tid] = n;
                            bar->top[tid] = mx;
                            bar->fl[tid] = first ? 0.0f : exp2_fast(was - n);
                            bar->fo[tid] = first ? 0.0f : exp2_fast((was - n) + static_cast<float>(X - xn));
                        }
                        X = xn;
                        wide |= look;
                        meet(false);
#pragma unroll
                        for (int r = 0; r < R; r++) {
                            m[r] = bar->n[r];
                            l[r] *= bar->fl[r];
                            f[r] = bar->fo[r];
                        }
                    } else {
#pragma unroll
                        for (int r = 0; r < R; r++) {
                            const float mn = fmaxf(m[r], over_warps(bar->red, r));
                            f[r] = m[r] == -INFINITY ? 0.0f : exp2_fast(m[r] - mn);
                            l[r] *= f[r];
                            m[r] = mn;
                        }
                    }
                    if (i > 0) {
                        tc_fence_after();
                        float o[Geo::NP];
                        tm_ld<Geo::NP>(o_col + lanes, o);
#pragma unroll
                        for (int c = 0; c < R * Geo::PT; c++) o[c] *= f[c % R];
#pragma unroll
                        for (int c = 0; c < Geo::NP; c += 16) tm_st16(o_col + lanes + c, reinterpret_cast<const uint32_t*>(o + c));
                        tm_wait_st();
                    }
                }
                // ---- weights, as the outputs' second operand ----
                wait(&bar->p_free[t & 1], ((t >> 1) & 1) ^ 1, 9);
                uint8_t* pw = smem + Geo::P_OFF + (t & 1) * Geo::P_STEP;
                const float vf = F8 ? exp2_fast(static_cast<float>(ve - X + kDecUnit)) : 1.0f;
#pragma unroll
                for (int r = 0; r < R; r += 2) {
                    float a = exp2_fast(s[r] - (m[r] == -INFINITY ? 0.0f : m[r]) + kBase);
                    float b = exp2_fast(s[r + 1] - (m[r + 1] == -INFINITY ? 0.0f : m[r + 1]) + kBase);
                    l[r] += a;
                    l[r + 1] += b;
                    if constexpr (F8) {
                        a *= vf;
                        b *= vf;
#pragma unroll
                        for (int k = 0; k < 3; k++) {
                            const unsigned c = split_e5m2(a, b);
                            const int n0 = k * R + r;
                            pw[dec_swizzle(128, n0, tid / 16) + tid % 16] = static_cast<uint8_t>(c);
                            pw[dec_swizzle(128, n0 + 1, tid / 16) + tid % 16] = static_cast<uint8_t>(c >> 8);
                        }
                    } else {
                        uint8_t* at = pw + (tid / 64) * Geo::NP * 128;
                        const int k = tid % 64;
                        auto put = [&](int n, unsigned c) {
                            *reinterpret_cast<uint16_t*>(at + dec_swizzle(128, n, k / 8) + (k % 8) * 2) = static_cast<uint16_t>(c);
                            *reinterpret_cast<uint16_t*>(at + dec_swizzle(128, n + 1, k / 8) + (k % 8) * 2) = static_cast<uint16_t>(c >> 16);
                        };
                        if constexpr (Geo::PT == 1) {
                            put(r, pack_bf16(a, b));
                        } else {
                            // the first term is cut off and the second a little larger than what is left: neither is zero or of
                            // the other sign, so that an infinite value stays one
                            const unsigned ha = __float_as_uint(a) & 0xffff0000u, hb = __float_as_uint(b) & 0xffff0000u;
                            put(r, ha >> 16 | hb);
                            put(R + r, pack_bf16(fmaf(a, 0x1p-20f, a - __uint_as_float(ha)), fmaf(b, 0x1p-20f, b - __uint_as_float(hb))));
                        }
                    }
                }
                fence_async_smem();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar->p_ready[t & 1]);
            }
            if (stop) break;
            // ---- the segment's outputs: thread d has dimension d of every row ----
            float o[Geo::NP];
            if (g.tiles > 0) {
                wait(&bar->p_free[(t - 1) & 1], ((t - 1) >> 1) & 1, 8);
                tc_fence_after();
                tm_ld<Geo::NP>(o_col + lanes, o);
            } else {
#pragma unroll
                for (int c = 0; c < Geo::NP; c++) o[c] = 0.0f;
            }
            if (meet(gone)) break;  // and the last maxima are read
            warp_reduce_multi<R>(l, lane);  // the lane's l[0] is the warp's sum of row reduce_index
            bar->red[warp][reduce_index<R>(lane, 0)] = l[0];
            if constexpr (F8) {
                const int x = __reduce_min_sync(0xffffffffu, low);
                const unsigned y = __ballot_sync(0xffffffffu, thin);
                if (lane == 0) bar->redx[warp] = y ? x - 256 : x;
            }
            meet(false);
            // Exponents, or all that a query row sees and the largest exponent, further apart than the weights can follow, scores past
            // what a reference holds beside them, or a reference raised by a row whose codes do not fill its exponent (an append
            // writes none): every row is done again below.
            bool lost = false;
            if constexpr (F8) {
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    const int x = bar->redx[w];
                    low = min(low, x < 0 ? x + 256 : x);
                    thin |= x < 0;
                }
                lost = X - low > (thin ? 8 : kDecSpread);
                for (int r = 0; wide && r < rows; r++)
                    lost |= bar->top[r] != -INFINITY && (fabsf(bar->top[r]) > 1048576.0f || (X > 0 && bar->T[r] < static_cast<float>(X - kDecSpread - 8)));
                v_item += 2 * g.tiles;
            }
            const int first = walk.deal.owner(g.pair_first), final_cta = walk.deal.owner(g.pair_end - 1);
            const int parts = final_cta - first + 1;
            float* my_part = ws.part + static_cast<int64_t>(2 * blockIdx.x + (g.lo == g.pair_first ? 1 : 0)) * ws.rows * PAD;
            bool odd = false;
#pragma unroll
            for (int r = 0; r < R; r++) {
                if (r >= rows) continue;
                float ls = bar->red[0][r] + bar->red[1][r] + bar->red[2][r] + bar->red[3][r];
                float x = o[r];
                if constexpr (!F8 && Geo::PT == 2) x += o[R + r];
                if constexpr (F8) x = (o[r] + o[R + r] + o[2 * R + r]) * power_of(-kDecUnit) * exp_byte(static_cast<unsigned>(X));
                if (parts == 1) {
                    x = vis[r] > 0 ? x / ls : 0.0f;
                    odd |= sq.n > 1 && tid < D && !(fabsf(x) <= 3.4e38f);
                    const __nv_bfloat16 v = __float2bfloat16_rn(x);
                    if (tid < D)
                        *reinterpret_cast<__nv_bfloat16*>(p.out + static_cast<int64_t>(sq.q0 + (row0 + r) / p.G) * p.out_stride +
                                                          static_cast<int64_t>(g.kvh * p.G + (row0 + r) % p.G) * D + tid) = v;
                } else {
                    float mx = m[r];
                    if (wide && mx != -INFINITY) {  // parts are joined by their largest scores
                        mx = bar->top[r];
                        const float back = exp2_fast(m[r] - mx);
                        x *= back;
                        ls *= back;
                    }
                    if (tid < D) my_part[r * PAD + tid] = x;
                    if (tid == 0)  // a sum below zero says that the range was passed
                        *reinterpret_cast<float2*>(my_part + r * PAD + D) = make_float2(mx, lost ? -1.0f : ls);
                }
            }
            if (parts > 1) {
                lost = false;  // the CTA that joins the parts learns it from them
                __threadfence();
                meet(false);
                if (tid == 0) {
                    unsigned* counter = ws.counters + first;  // a CTA starts at most one (sequence, kv head) that it does not end
                    const bool last = atomicAdd(counter, 1u) == static_cast<unsigned>(parts - 1);
                    if (last) *counter = 0u;
                    bar->last = last;
                }
                meet(false);
                if (bar->last) {
                    __threadfence();
                    auto part_of = [&](int i) {
                        // the first CTA's blocks of the pair are its last segment unless the pair starts it
                        return ws.part + static_cast<int64_t>(2 * (first + i) + (i == 0 ? 1 : 0)) * ws.rows * PAD;
                    };
                    for (int q = tid; q < rows * (D / 4); q += kDecSoft) {
                        const int r = q / (D / 4), d = (q % (D / 4)) * 4, token = (row0 + r) / p.G;
                        // sixteen parts' loads under way at once: a pass over them is a few trips to L2
                        float M = -INFINITY, ls = 0.0f;
                        float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        for (int i0 = 0; i0 < parts; i0 += 16) {
                            float2 ml[16];
                            float4 v[16];
                            float mn = M;
#pragma unroll
                            for (int i = 0; i < 16; i++) {
                                const float* pr = part_of(i0 + i) + r * PAD;
                                const bool in = i0 + i < parts;
                                ml[i] = in ? __ldcg(reinterpret_cast<const float2*>(pr + D)) : make_float2(-INFINITY, 0.0f);
                                v[i] = in ? __ldcg(reinterpret_cast<const float4*>(pr + d)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            }
#pragma unroll
                            for (int i = 0; i < 16; i++) mn = fmaxf(mn, ml[i].x);
                            const float b0 = mn == -INFINITY ? 0.0f : mn;
                            const float c = exp2_fast(M - b0);
                            M = mn;
                            ls *= c;
                            a.x *= c, a.y *= c, a.z *= c, a.w *= c;
#pragma unroll
                            for (int i = 0; i < 16; i++) {
                                const float f = exp2_fast(ml[i].x - b0);
                                lost |= ml[i].y < 0.0f;
                                a.x = fmaf(f, v[i].x, a.x), a.y = fmaf(f, v[i].y, a.y), a.z = fmaf(f, v[i].z, a.z), a.w = fmaf(f, v[i].w, a.w);
                                ls = fmaf(f, ml[i].y, ls);
                            }
                        }
                        const bool sees = sq.len > 0 && sq.len - sq.n + token >= 0;
                        const float inv = 1.0f / ls;
                        a = sees ? make_float4(a.x * inv, a.y * inv, a.z * inv, a.w * inv) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        odd |= sq.n > 1 && !(fabsf(a.x) + fabsf(a.y) + fabsf(a.z) + fabsf(a.w) <= 3.4e38f);
                        *reinterpret_cast<uint2*>(p.out + static_cast<int64_t>(sq.q0 + token) * p.out_stride +
                                                  static_cast<int64_t>(g.kvh * p.G + row0 + r - token * p.G) * D + d) =
                            make_uint2(pack_bf16(a.x, a.y), pack_bf16(a.z, a.w));
                    }
                }
            }
            // A value that is not finite, behind some row's mask, reaches that row as 0 * inf through the products (a single new
            // token sees everything): where there is one, and where the weights' range was passed, every row is done again in
            // plain loops over what it sees.
            bool redo = meet(odd || lost);
            if (redo && !meet(lost))
                redo = odd_values<KIND, D>(p, g.b, sq.q0, g.kvh, max(0, min(sq.len, sq.len - sq.n + row0 / p.G + 1)), sq.len, lane);
            if (redo) {
                for (int r = warp; r < rows; r += 4) {
                    const int token = (row0 + r) / p.G, head = g.kvh * p.G + row0 + r - token * p.G;
                    const int see = max(0, min(sq.len, sq.len - sq.n + token + 1));
                    float mm, ll, a[D / 32];
                    attend_row<KIND, D>(p, g.b, sq.q0, sq.q0 + token, head, 0, see, lane, &bar->beat, mm, ll, a);
                    uint16_t* to = p.out + static_cast<int64_t>(sq.q0 + token) * p.out_stride + static_cast<int64_t>(head) * D + lane * (D / 32);
                    const float inv = see > 0 ? 1.0f / ll : 0.0f;
#pragma unroll
                    for (int i = 0; i < D / 32; i += 2) *reinterpret_cast<unsigned*>(to + i) = pack_bf16(a[i] * inv, a[i + 1] * inv);
                }
            }
            tc_fence_before();
        }
    }
    __syncthreads();
    if (warp == 4) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 128;" ::"r"(tmem) : "memory");
    }
}

}  // namespace oomb
