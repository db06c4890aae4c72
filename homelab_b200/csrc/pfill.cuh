// pfill.cuh - causal grouped-query attention of many new tokens (prefill chunks over a paged
// cache, whole prompts over their own rows) on the 5th-generation tensor cores.
//
// A tile is 2 x 128 query rows of one kv head: row r of a half is new token r / G, query
// head r % G of the group, so a group's heads share every key and value that is loaded
// (floor(128 / G) tokens a half).  Per 128 positions and half, with S and O in tensor memory:
//   S = Q K^T          tcgen05.mma, both operands in shared memory (TMA, 128-byte swizzle)
//   P = e^(S - m)      one thread per row, fp32, rounded to bf16 and written over S
//   O += P V           tcgen05.mma, P from tensor memory
// m is the running maximum; O is multiplied up only when m has grown by more than 2^8 (the
// factor cancels in O / l, and e^8 in base 2 keeps bf16 and fp32 far from overflow), which after
// the first tiles is rare.
//
// Bound: with D = 128 a pair of halves costs 32 products of 64 tensor-pipe cycles per 128
// positions (a product of M = 128 takes about 64 cycles for any N up to 128: its operands come
// out of shared memory) and 2 x 16,384 exponentials, which at 16 a cycle and SM are 2,048 cycles as
// well.  The two halves run in turn: while one's scores go through the exponentials,
// the tensor cores multiply the other's.  One issuing warp orders the products
//   S0 S1 | O0 S0' | O1 S1' | ...,
// and since they complete in order, the barrier of S0' also says that O0 is at rest, so a
// row's thread may rescale it without another wait, and S may be overwritten as soon as
// P was consumed.  Scores, maxima, exponentials and products of one half still follow one
// another (tensor memory has no room for second scores beside two outputs of 128 columns), which leaves
// the tensor pipe active 58 % of the time.  Prompts of 8,192 and 3,001 tokens
// (32 heads over 8, D = 128) take 515-524 us, 1,190-1,210 TFLOP/s, in short bursts, and 608 us, 1,026, called on end for a
// second, when the power limit lowers the clock.
// Tried when this stood at 569 us, and no faster: two threads a row (619 us), scores of 64 positions at a time, made
// ahead (633 us: the products cost the same at N = 64).
//
// Warps: 0-3 and 4-7 the softmax of half 0 and 1 (and their epilogue), one thread a row;
// 8 issues the products (and zeroes value rows behind the last position, which may hold
// anything: 0 * NaN); 9 loads by TMA through a ring of key and value tiles, page by page for a
// paged cache (a page of 16 or more rows keeps the swizzle's 8-row pattern); for an e4m3 cache 12-15
// turn the loaded codes into bf16 tiles on the way (once per tile, for all 256 rows).
//
// Work: plan_kernel lists the units (a tile, or a part of its positions when there are too few
// tiles to fill the SMs), longest first; a CTA takes the next when it is through with one.  Parts leave (acc, m, l) in the
// workspace, joined in order by join_kernel.  Every wait is bounded.
#pragma once

#include "pattn.cuh"
#include "tcptx.cuh"

namespace oomb {

constexpr int kFaTile = 128;
constexpr int kFaRows = 256;       // rows of a tile pair
// Parts of a tile's weights that are handed to the product on their own; measured on two packed prompts of 8192 and 3001
// tokens (32 heads over 8, D = 128): one part 610 us, two 569-600, four 601-625 (each hand-over waits for its stores).
constexpr int kFaParts = 2;
constexpr int kFaSoft = 8;         // softmax warps
// Weights are made, and summed, as 2^-8 of what they are: with the 2^8 that a row's maximum may lag behind they are one at most,
// and no product with a value passes what fp32 holds that the value itself does not.  (Those below 2^-118 of the row's largest
// are zero, where fp32's own range would end at 2^-126.)
constexpr float kFaDown = 8.0f;
constexpr int kFaMinPart = 4;      // key tiles of a part at least
constexpr int kPlanThreads = 256;
constexpr int kPlanBuckets = 512;
constexpr int kPlanSeqs = 1024;    // sequences whose numbers are kept in shared memory

enum : unsigned {
    ERR_FA_WAIT = 0xa00,  // a prefill pipeline wait ran out (+ the waiting role)
};

struct __align__(16) FaUnit {
    Seq s;
    int b, i0;     // sequence, first new token (of the sequence)
    int kv0, kv1;  // key tiles
    int slot;      // partial outputs' slot, or -1: the unit is its tile's only one
};
struct __align__(16) FaSplit {
    Seq s;
    int i0, b, slot, parts, pad;
};
static_assert(sizeof(FaUnit) == 32 && sizeof(FaSplit) == 32, "read as two int4");
struct FaHead {
    int units, splits, slots;
    int next;  // units dealt out beyond the CTAs' first
};

struct FaWs {
    FaHead* head;
    FaUnit* units;
    FaSplit* splits;
    float* part;  // [slot][kv head][256][fa_line(D)]: acc, m, l
    int max_units, max_slots, sms;
    int direct;  // few sequences and tiles: every CTA plans by itself
};

// Floats of a partial row: acc, m, l, 32-byte aligned.
__host__ __device__ constexpr int fa_line(int D) { return D + 8; }

// Tokens of a half tile.
__host__ __device__ inline int fa_tokens(int G) { return kFaTile / G; }

__device__ __forceinline__ int fa_tiles_of(const Seq& s, int tq) { return (s.n + 2 * tq - 1) / (2 * tq); }
// Key tiles that the tokens [i0, i1) of a sequence see together.
__device__ __forceinline__ int fa_key_tiles(const Seq& s, int i1) {
    const int vis = max(0, min(s.len, s.len - s.n + min(i1, s.n)));
    return (vis + kFaTile - 1) / kFaTile;
}

// When the last CTA should finish, in key tiles, with parts of `len` at most: with at most a unit an SM that is the
// longest unit, else (the longest go first) the share and half of the shortest; writing and joining parts costs about
// two.
__device__ __forceinline__ int fa_cost(int longest, int shortest, int share, int len, int units, int sms) {
    const int parts = (longest + len - 1) / len, unit = (longest + parts - 1) / parts;
    return (units <= sms ? unit : max(unit, share + min(unit, shortest) / 2)) + (parts > 1 ? 2 : 0);
}

// One CTA.  The sequences' numbers are read once (up to kPlanSeqs of them) and a warp takes a sequence, a lane a
// tile.  Up to as many units as SMs are listed as they come; more are sorted by a counting sort on their length.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const __grid_constant__ PattnParams p, const __grid_constant__ FaWs ws) {
    __shared__ int hist[kPlanBuckets];
    __shared__ Seq seqs[kPlanSeqs];
    __shared__ unsigned long long total_s;
    __shared__ int slots_s, splits_s, units_s, longest_s, shortest_s, count_s[6], warp_sum[32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = kPlanThreads / 32;
    if (tid == 0) {
        total_s = 0;
        slots_s = splits_s = units_s = longest_s = 0;
        shortest_s = 1 << 30;
        for (int k = 0; k < 6; k++) count_s[k] = 0;
    }
    for (int i = tid; i < kPlanBuckets; i += kPlanThreads) hist[i] = 0;
    pdl_wait();
    pdl_launch_dependents();
    const int tq = fa_tokens(p.G);
    auto read = [&](int b, unsigned* err) {
        Seq s = read_seq(p.q_start, p.kv_len, b, p.T, p.kv_max, err);
        if (s.n > p.max_q) {
            record_error(err, ERR_KV_SEQ);
            s.n = 0;
        }
        return s;
    };
    for (int b = tid; b < p.B; b += kPlanThreads) {
        const Seq s = read(b, p.err);
        if (b < kPlanSeqs) seqs[b] = s;
    }
    __syncthreads();
    auto seq_of = [&](int b) { return b < kPlanSeqs ? seqs[b] : read(b, nullptr); };
    unsigned long long work = 0;
    int longest = 1, shortest = 1 << 30;
    for (int b = warp; b < p.B; b += warps) {
        const Seq s = seq_of(b);
        const int nt = fa_tiles_of(s, tq);
        for (int i = lane; i < nt; i += 32) {
            const int keys = max(1, fa_key_tiles(s, (i + 1) * 2 * tq));
            work += keys;
            longest = max(longest, keys);
            shortest = min(shortest, keys);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) work += __shfl_xor_sync(0xffffffffu, work, o);
    longest = __reduce_max_sync(0xffffffffu, longest);
    shortest = __reduce_min_sync(0xffffffffu, shortest);
    if (lane == 0 && work) {
        atomicAdd(&total_s, work);
        atomicMax(&longest_s, longest);
        atomicMin(&shortest_s, shortest);
    }
    __syncthreads();
    // How long a part may be: an SM's even share of the step or more (so that there are at most two parts an SM), or a whole
    // tile.  Of a few lengths the one whose last CTA should finish first.
    const unsigned long long share64 = (total_s * p.Hkv + ws.sms - 1) / ws.sms;
    const int share = share64 > (1u << 24) ? (1 << 24) : max(kFaMinPart, static_cast<int>(share64));
    longest = longest_s;
    int chunk = longest;
    if (longest > share) {
        // lane k tries the k-th length: 1, 1 1/8, 1 1/4, 1 1/2, 2 shares, a whole tile
        const int eighths = lane == 0 ? 8 : lane == 1 ? 9 : lane == 2 ? 10 : lane == 3 ? 12 : 16;
        const int len = lane < 5 ? (share * eighths + 7) / 8 : longest;
        int units = 0;
        for (int b = warp; b < p.B; b += warps) {
            const Seq s = seq_of(b);
            const int nt = fa_tiles_of(s, tq);
#pragma unroll 1
            for (int i = 0; i < nt; i++) units += (max(1, fa_key_tiles(s, (i + 1) * 2 * tq)) + len - 1) / len;
        }
        if (lane < 6 && units) atomicAdd(&count_s[lane], units);
        __syncthreads();
        const int cost = fa_cost(longest, shortest_s, share, len, count_s[min(lane, 5)] * p.Hkv, ws.sms);
        const int best = __reduce_min_sync(0xffffffffu, lane < 6 ? cost : 1 << 30);
        chunk = __shfl_sync(0xffffffffu, len, __ffs(__ballot_sync(0xffffffffu, lane < 6 && cost == best)) - 1);
    }
    auto parts_of = [&](int keys) { return max(1, (keys + chunk - 1) / chunk); };
    // lengths up to 128 apart, longer ones to a sixteenth
    auto bucket_of = [&](int k) {
        const int e = 31 - __clz(max(k, 1));
        return kPlanBuckets - 1 - (k < 128 ? k : min(128 + (e - 7) * 16 + ((k >> (e - 4)) & 15), kPlanBuckets - 1));
    };
    // how many units, and of what length
    int mine = 0;
    for (int b = warp; b < p.B; b += warps) {
        const Seq s = seq_of(b);
        const int nt = fa_tiles_of(s, tq);
        for (int i = lane; i < nt; i += 32) {
            const int keys = fa_key_tiles(s, (i + 1) * 2 * tq), parts = parts_of(keys);
            mine += parts;
            // a tile's parts differ by one key tile at most
            const int each = keys / parts, more = keys - each * parts;
            if (more) atomicAdd(&hist[bucket_of(each + 1)], more);
            atomicAdd(&hist[bucket_of(each)], parts - more);
        }
    }
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0 && mine) atomicAdd(&units_s, mine);
    __syncthreads();
    const int units = units_s;
    // more units than the workspace holds: only sequences that overlap each other make so many
    if (units > ws.max_units) {
        if (tid == 0) {
            record_error(p.err, ERR_KV_SEQ);
            *ws.head = FaHead{};
        }
        return;
    }
    const bool sorted = units * p.Hkv > ws.sms;
    if (sorted) {  // where each length's units begin, the longest first
        static_assert(kPlanBuckets == 2 * kPlanThreads, "two buckets a thread");
        const int v0 = hist[2 * tid], v = v0 + hist[2 * tid + 1];
        int inc = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += u;
        }
        if (lane == 31) warp_sum[warp] = inc;
        __syncthreads();
        int before = 0;
        for (int w = 0; w < warp; w++) before += warp_sum[w];
        hist[2 * tid] = before + inc - v;
        hist[2 * tid + 1] = before + inc - v + v0;
    } else if (tid == 0) {
        hist[0] = 0;
    }
    __syncthreads();
    for (int b = warp; b < p.B; b += warps) {
        const Seq s = seq_of(b);
        const int nt = fa_tiles_of(s, tq);
        for (int i = lane; i < nt; i += 32) {
            const int keys = fa_key_tiles(s, (i + 1) * 2 * tq), parts = parts_of(keys);
            int slot = -1;
            if (parts > 1) {
                slot = atomicAdd(&slots_s, parts);
                ws.splits[atomicAdd(&splits_s, 1)] = FaSplit{s, i * 2 * tq, b, slot, parts, 0};
            }
            const int each = keys / parts, more = keys - each * parts;
            for (int j = 0; j < parts; j++) {
                const int k0 = j * each + min(j, more), k1 = k0 + each + (j < more ? 1 : 0);
                const int at = atomicAdd(&hist[sorted ? bucket_of(k1 - k0) : 0], 1);
                FaUnit u;
                u.s = s;
                u.b = b;
                u.i0 = i * 2 * tq;
                u.kv0 = k0;
                u.kv1 = k1;
                u.slot = slot < 0 ? -1 : slot + j;
                ws.units[at] = u;
            }
        }
    }
    __syncthreads();
    if (tid == 0) *ws.head = FaHead{units, splits_s, slots_s, 0};
}

// ---- PTX ------------------------------------------------------------------------------

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
            smem_addr(dst)),
        "l"(map), "r"(smem_addr(bar)), "r"(x), "r"(y), "r"(z)
        : "memory");
}
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
            smem_addr(dst)),
        "l"(map), "r"(smem_addr(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// bf16 x bf16 -> fp32, M = 128: A and B in shared memory (B K-major), or A in tensor memory and B MN-major.
__host__ __device__ constexpr uint32_t fa_idesc(int n, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24);
}
// Descriptors by their low words and a common high word.
__device__ __forceinline__ void fa_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t hi, uint32_t idesc, int acc) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 da, db;\n setp.ne.b32 p, %5, 0;\n mov.b64 da, {%1, %3};\n mov.b64 db, {%2, %3};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n}" ::"r"(d),
        "r"(a), "r"(b), "r"(hi), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void fa_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t hi, uint32_t idesc, int acc) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 db;\n setp.ne.b32 p, %5, 0;\n mov.b64 db, {%2, %3};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n}" ::"r"(d),
        "r"(a), "r"(b), "r"(hi), "r"(idesc), "r"(acc)
        : "memory");
}
// An MN-major operand in the 128-byte swizzle: rows of 64 values (128 bytes) along N, 8-row groups along K 1024
// bytes apart (stride offset), further 64-value columns `lead` bytes apart (leading offset).
__host__ __device__ constexpr uint64_t fa_desc_mn(uint32_t addr, uint32_t lead) {
    return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(lead >> 4) << 16) | (64ull << 32) | (1ull << 46) |
           (2ull << 61);
}

__device__ __forceinline__ void tm_ld32(uint32_t taddr, float* v) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tm_ld16(uint32_t taddr, float* v) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tm_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
// 32 bytes (32-byte aligned): a thread that owns a row writes whole sectors, in half the trips of 16-byte stores.
__device__ __forceinline__ void st_global_v8(void* p, const uint32_t (&r)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                 "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ---- shared memory --------------------------------------------------------------------

template <int KIND, int D>
struct FaGeo {
    static constexpr bool F8 = KIND == KV_E4M3;
    static constexpr int TILE = kFaTile * D * 2;         // bytes of 128 rows in bf16
    static constexpr int HALF = kFaTile * 128;           // bytes of 64 columns of them
    static constexpr int CODES = kFaTile * D;            // bytes of 128 rows in e4m3
    static constexpr int RAW = F8 ? 2 : 0;               // slots of codes before their conversion
    static constexpr int ROOM = 224 * 1024 - 2 * TILE - RAW * CODES;
    static constexpr int STAGES = ROOM / TILE < 8 ? ROOM / TILE : 8;
    static constexpr int Q_OFF = 0;
    static constexpr int KV_OFF = 2 * TILE;
    static constexpr int RAW_OFF = KV_OFF + STAGES * TILE;
    static constexpr int EXP_OFF = RAW_OFF + RAW * CODES;
    static constexpr int BAR_OFF = EXP_OFF + RAW * kFaTile;
    static constexpr int TOTAL = BAR_OFF + 448;
    // registers: the softmax threads hold a row of scores; the rest give theirs up (the sums equal the launch's)
    static constexpr int THREADS = kFaSoft * 32 + (F8 ? 256 : 128);
    static constexpr int SOFT_REGS = F8 ? 192 : 208;
    static constexpr int REST_REGS = F8 ? 64 : 88;
    static_assert(kFaSoft * 32 * SOFT_REGS + (THREADS - kFaSoft * 32) * REST_REGS <= THREADS * (F8 ? 128 : 168), "register split");
    static_assert(TOTAL <= 227 * 1024, "shared memory");
};

struct FaBars {
    uint64_t q_full[2], q_empty, s_full[2], p_ready[2][kFaParts], o_full[2], kv_full[8], kv_empty[8], raw_full[2], raw_empty[2], u_full[2], u_empty[2], done;
    uint32_t tmem;
    unsigned beat;  // moves while rows are done again
    int kvh[2];  // the CTA's current and next unit: kv head (-1: no more), and the rest
    __align__(16) FaUnit unit[2];
};

// The value of lane 0 in every lane: the compiler then keeps it, and what it makes of it, in uniform
// registers, which the tensor instructions take their descriptors from.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ bool elect_one() {
    unsigned r;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(r));
    return r != 0;
}

// A role's pipeline position over a ring of N stages.
template <int N>
struct Ring {
    int i = 0;
    unsigned phase = 0;
    __device__ void next() {
        if (++i == N) {
            i = 0;
            phase ^= 1;
        }
    }
};

// The larger of three (one instruction on sm_100).
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// 2^x of two values on the FMA units: x = r + f, r the nearest integer, 2^f by a polynomial of degree 4
// fitted to it on [-1/2, 1/2] (Remez exchange on the relative error: 2.7e-6, an 800th of the weights'
// rounding to bf16), r added to the exponent.  Below -126 it is 0, as a hidden position's weight has to be, and NaN is NaN
// (the larger of x and 0 is that, where x is not at least -126).  x < 128.
__device__ __forceinline__ float2 exp2_fma(float2 x) {
    constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23: adding it rounds to an integer
    const bool in_x = x.x >= -126.0f, in_y = x.y >= -126.0f;
    float2 out;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(out.x) : "f"(x.x), "f"(0.0f));
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(out.y) : "f"(x.y), "f"(0.0f));
    const float2 one = make_float2(1.0f, 1.0f);
    const float2 t = ffma2(x, one, make_float2(kMagic, kMagic));
    const float2 r = ffma2(t, one, make_float2(-kMagic, -kMagic));
    const float2 f = ffma2(r, make_float2(-1.0f, -1.0f), x);
    float2 y = ffma2(make_float2(9.570102207e-03f, 9.570102207e-03f), f, make_float2(5.591785908e-02f, 5.591785908e-02f));
    y = ffma2(y, f, make_float2(2.402474433e-01f, 2.402474433e-01f));
    y = ffma2(y, f, make_float2(6.931217909e-01f, 6.931217909e-01f));
    y = ffma2(y, f, make_float2(9.999992847e-01f, 9.999992847e-01f));
    return make_float2(in_x ? __int_as_float(__float_as_int(y.x) + (__float_as_int(t.x) << 23)) : out.x,
                       in_y ? __int_as_float(__float_as_int(y.y) + (__float_as_int(t.y) << 23)) : out.y);
}

// As mbar_wait, but the clock and the limit (a load from global memory, some 600 cycles) are read only
// after many polls: a wait of a tile's length must not pay for them.  While `beat` moves a warp of the CTA does rows again
// (attend_row), which takes as long as it takes, and the limit begins anew.
__device__ __forceinline__ bool fa_wait_lane(uint64_t* bar, unsigned parity, unsigned* err, unsigned code, const unsigned* beat) {
    for (int i = 0; i < 64; i++)
        if (mbar_try_wait(bar, parity)) return true;
    const volatile unsigned* at = beat;
    unsigned long long t0 = global_ns();
    const unsigned long long limit = wait_limit();
    unsigned seen = *at;
    for (;;) {
        if (mbar_try_wait(bar, parity)) return true;
        const unsigned long long now = global_ns();
        if (now - t0 <= limit) continue;
        const unsigned b = *at;
        if (b == seen) {
            record_error(err, code);
            return false;
        }
        seen = b;
        t0 = now;
    }
}
// The same for a warp whose lanes agree: where one gave up all do, since what follows (tensor memory, votes, the end of the
// role) takes the warp together.  The warps that pace the products go on after a wait that ran out, over whatever is in their
// tiles, and agree once a tile (two packed prompts of 8,192 and 3,001 tokens took 524 us without agreeing, 530 with a vote a
// wait, 527 so).
__device__ __forceinline__ bool fa_wait(uint64_t* bar, unsigned parity, unsigned* err, unsigned code, const unsigned* beat) {
    return __all_sync(0xffffffffu, fa_wait_lane(bar, parity, err, code, beat));
}
// The waits at a CTA's end for copies and products under way, which end by themselves: the limit that a caller may shorten does
// not count here, since a CTA that left before them would have its shared memory written after it.
__device__ __forceinline__ void fa_drain(uint64_t* bar, unsigned parity, unsigned* err, unsigned code) {
    if (mbar_try_wait(bar, parity)) return;
    const unsigned long long t0 = global_ns();
    while (!mbar_try_wait(bar, parity))
        if (global_ns() - t0 > kWaitLimitNs) {
            record_error(err, code);
            return;
        }
}

// The plan of up to 32 sequences with up to 32 tiles together, by one warp and without a launch of its own (which takes four
// us of a step of short prompts or drafts): lane i keeps tile i.
struct FaTiles {
    Seq s;
    int b, i0, keys, parts;  // the lane's tile
    int first, slot;         // its first unit, its first slot
    int units;
    // The two halves (lanes 0 and 1) of unit v's record.
    __device__ __forceinline__ int4 unit(int v, int lane) const {
        const int t = min(31, __popc(__ballot_sync(0xffffffffu, first + parts <= v)));
        auto of = [&](int x) { return __shfl_sync(0xffffffffu, x, t); };
        const int j = v - of(first), k = of(keys), n = max(1, of(parts)), each = k / n, more = k - each * n;
        const int k0 = j * each + min(j, more);
        const int4 lo = make_int4(of(s.q0), of(s.n), of(s.len), of(b));
        const int4 hi = make_int4(of(i0), k0, k0 + each + (j < more ? 1 : 0), n > 1 ? of(slot) + j : -1);
        return lane == 0 ? lo : hi;
    }
};

// (Its arguments come by value: a reference to the kernel's parameters would be read through the caches.)
__device__ __noinline__ FaTiles fa_plan_tiles(const int32_t* q_start, const int32_t* kv_len, int B, int T, int kv_max, int max_q, int Hkv,
                                              int sms, int tq, int lane, FaSplit* splits, FaHead* head, unsigned* err) {
    Seq s{};
    if (lane < B) {
        s = read_seq(q_start, kv_len, lane, T, kv_max, err);
        if (s.n > max_q) {
            record_error(err, ERR_KV_SEQ);
            s.n = 0;
        }
    }
    auto scan = [&](int v) {  // inclusive
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        return v;
    };
    const int mine = lane < B ? fa_tiles_of(s, tq) : 0, ends = scan(mine);
    int tiles = __shfl_sync(0xffffffffu, ends, 31);
    if (tiles > 32) {  // only sequences that overlap each other make so many
        record_error(err, ERR_KV_SEQ);
        tiles = 0;
    }
    FaTiles t{};
    for (int k = 0; k < B; k++) t.b += __shfl_sync(0xffffffffu, ends, k) <= lane;
    t.b = min(t.b, 31);
    t.s.q0 = __shfl_sync(0xffffffffu, s.q0, t.b);
    t.s.n = __shfl_sync(0xffffffffu, s.n, t.b);
    t.s.len = __shfl_sync(0xffffffffu, s.len, t.b);
    const bool has = lane < tiles;
    t.i0 = (lane - __shfl_sync(0xffffffffu, ends - mine, t.b)) * 2 * tq;
    t.keys = has ? fa_key_tiles(t.s, t.i0 + 2 * tq) : 0;
    const int work = has ? max(1, t.keys) : 0;
    // (a 64-bit division would take longer than the rest; 2^28 tiles at most, and the slots have room for a share off by 2^-22)
    const float even = static_cast<float>(__reduce_add_sync(0xffffffffu, work)) * Hkv * (1.0f / sms);
    const int share = max(kFaMinPart, static_cast<int>(fminf(ceilf(even), 16777216.0f)));
    const int longest = max(1, __reduce_max_sync(0xffffffffu, work)), shortest = __reduce_min_sync(0xffffffffu, has ? work : 1 << 30);
    int chunk = longest;
    if (longest > share) {  // as plan_kernel chooses
        // lane k keeps the k-th length's units and its cost
        const int eighths = lane == 0 ? 8 : lane == 1 ? 9 : lane == 2 ? 10 : lane == 3 ? 12 : 16;
        const int len = lane < 5 ? (share * eighths + 7) / 8 : longest;
        int units = 0;
#pragma unroll 1
        for (int k = 0; k < 6; k++) {
            const int of = __shfl_sync(0xffffffffu, len, k), sum = __reduce_add_sync(0xffffffffu, (work + of - 1) / of);
            units = lane == k ? sum : units;
        }
        const int cost = fa_cost(longest, shortest, share, len, units * Hkv, sms);
        const int best = __reduce_min_sync(0xffffffffu, lane < 6 ? cost : 1 << 30);
        chunk = __shfl_sync(0xffffffffu, len, __ffs(__ballot_sync(0xffffffffu, lane < 6 && cost == best)) - 1);
    }
    t.parts = has ? (work + chunk - 1) / chunk : 0;
    // units in the low half, slots in the high one (no more than 32 and twice the SMs)
    const int split = t.parts > 1 ? t.parts : 0, both = t.parts | split << 16, ue = scan(both);
    t.first = (ue - both) & 0xffff;
    t.slot = (ue - both) >> 16;
    t.units = __shfl_sync(0xffffffffu, ue, 31) & 0xffff;
    if (blockIdx.x == 0) {  // for the join
        const unsigned m = __ballot_sync(0xffffffffu, split > 0);
        if (split) splits[__popc(m & ((1u << lane) - 1))] = FaSplit{t.s, t.i0, t.b, t.slot, t.parts, 0};
        if (lane == 0) head->splits = __popc(m);
    }
    return t;
}

// What every role derives from a unit: the sequence and each half's key tiles.
struct FaWork {
    Seq s;
    int b, i0, kvh, kv0, keys;  // keys: tiles of the unit
    int nh[2];                  // tiles that half h multiplies (the first of the unit's)
    int slot;
    int base;                   // packed rows: the sequence's first
};

__device__ __forceinline__ FaWork fa_work(const PattnParams& p, const FaUnit& u, int kvh, int tq) {
    FaWork w;
    w.s = u.s;
    w.b = u.b;
    w.i0 = u.i0;
    w.kv0 = u.kv0;
    w.keys = u.kv1 - u.kv0;
    w.slot = u.slot;
    w.kvh = kvh;
    w.base = p.kv.seq_rows ? w.b * p.kv.seq_rows : w.s.q0;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int i = w.i0 + h * tq;
        w.nh[h] = i < w.s.n ? max(0, min(w.keys, fa_key_tiles(w.s, i + tq) - w.kv0)) : 0;
    }
    return w;
}

// Values that are not finite, behind some row's mask, reach that row as 0 * inf through the products: the rows `again` of a
// warp (a lane's token, head, positions seen and partial row are its own) are done again in plain loops over what they see of
// the positions [j0, j1) that were multiplied, if there is such a value (else what they see is not finite).
template <int KIND, int D>
__device__ __noinline__ void fa_redo(const PattnParams& p, int b, int base, int kvh, int j0, int j1, unsigned again, int token, int head, int vis,
                                     float* line, int lane, unsigned* beat) {
    const bool mine = again >> lane & 1;
    const int hidden = __reduce_min_sync(0xffffffffu, mine ? max(vis, j0) : j1);
    if (!odd_values<KIND, D>(p, b, base, kvh, hidden, j1, lane)) return;
    while (again) {
        const int src = __ffs(again) - 1;
        again &= again - 1;
        const int tk = __shfl_sync(0xffffffffu, token, src), hd = __shfl_sync(0xffffffffu, head, src), see = __shfl_sync(0xffffffffu, vis, src);
        float* const to = reinterpret_cast<float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(line), src));
        float mm, ll, a[D / 32];
        attend_row<KIND, D>(p, b, base, tk, hd, j0, min(see, j1), lane, beat, mm, ll, a);
        if (to == nullptr) {
            uint16_t* o = p.out + static_cast<int64_t>(tk) * p.out_stride + static_cast<int64_t>(hd) * D + lane * (D / 32);
            const float iv = see > 0 ? 1.0f / ll : 0.0f;
#pragma unroll
            for (int e = 0; e < D / 32; e += 2) {
                const __nv_bfloat162 b2 = __floats2bfloat162_rn(a[e] * iv, a[e + 1] * iv);
                *reinterpret_cast<__nv_bfloat162*>(o + e) = b2;
            }
        } else {
#pragma unroll
            for (int e = 0; e < D / 32; e++) to[lane * (D / 32) + e] = a[e];
            if (lane == 0) *reinterpret_cast<float2*>(to + D) = make_float2(mm - kFaDown, ll);
        }
    }
}

template <int KIND, int D>
__global__ void __launch_bounds__(FaGeo<KIND, D>::THREADS, 1)
    fa_kernel(const __grid_constant__ PattnParams p, const __grid_constant__ FaWs ws, const __grid_constant__ CUtensorMap qmap,
              const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    using Geo = FaGeo<KIND, D>;
    constexpr bool F8 = Geo::F8;
    constexpr int ST = Geo::STAGES, CH = D / 64;  // 64-column chunks of a tile
    extern __shared__ __align__(1024) uint8_t smem[];
    FaBars* bar = reinterpret_cast<FaBars*>(smem + Geo::BAR_OFF);
    static_assert(sizeof(FaBars) <= Geo::TOTAL - Geo::BAR_OFF, "barriers");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int tq = fa_tokens(p.G);

    if (smem_addr(smem) & 1023u) {  // the swizzle's pattern starts there
        if (tid == 0) record_error(p.err, ERR_FA_WAIT + 15);
        return;
    }
    if (tid == 0) {
        for (int h = 0; h < 2; h++) {
            mbar_init(&bar->q_full[h], 1);
            mbar_init(&bar->s_full[h], 1);
            for (int part = 0; part < kFaParts; part++) mbar_init(&bar->p_ready[h][part], 4);
            mbar_init(&bar->o_full[h], 1);
        }
        mbar_init(&bar->q_empty, 1);
        mbar_init(&bar->done, 1);
        bar->beat = 0;
        for (int i = 0; i < ST; i++) {
            mbar_init(&bar->kv_full[i], F8 ? 4 : 1);
            mbar_init(&bar->kv_empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&bar->u_full[i], 1);
            mbar_init(&bar->u_empty[i], kFaSoft + 1 + (F8 ? 4 : 0));
            mbar_init(&bar->raw_full[i], 1);
            mbar_init(&bar->raw_empty[i], 4);
        }
        fence_barrier_init();
    }
    if (warp == kFaSoft) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&bar->tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bar->tmem;
    pdl_wait();
    pdl_launch_dependents();
    // The loader deals the CTA its units (the first by its index, then whichever is next) and tells the other warps.
    Ring<2> feed;
    auto take = [&](FaWork& w) {
        if (!fa_wait(&bar->u_full[feed.i], feed.phase, p.err, ERR_FA_WAIT + 12, &bar->beat)) return false;
        const int kvh = *static_cast<volatile int*>(&bar->kvh[feed.i]);
        if (kvh >= 0) w = fa_work(p, bar->unit[feed.i], kvh, tq);
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar->u_empty[feed.i]);
        feed.next();
        return kvh >= 0;
    };
    // the register split stands inside the roles' branches: behind a join the smaller share would bind them all
    if (warp < kFaSoft) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Geo::SOFT_REGS));
        // ---- softmax and epilogue: one thread per row ----
        const int h = warp >> 2, row = tid & 127;
        const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lane_base + h * 128, to = tmem + lane_base + 256 + h * 128;
        unsigned s_ph = 0, o_ph = 0;
        bool ok = true;
        // a scale below zero turns the scores' sign, and one of zero makes them zero (before the mask: 0 * -inf is NaN)
        const float scale = p.scale_log2 == 0.0f ? 1.0f : fabsf(p.scale_log2);
        for (FaWork w; ok && take(w);) {
            const int token_of = row / p.G, head_of = row - token_of * p.G;
            const int token = w.i0 + h * tq + token_of;
            const bool valid = token_of < tq && token < w.s.n;
            const int vis = valid ? max(0, min(w.s.len, w.s.len - w.s.n + token + 1)) : 0;
            float m = -INFINITY, l = 0.0f;
            for (int i = 0; i < w.nh[h]; i++) {
                const bool there = fa_wait_lane(&bar->s_full[h], s_ph, p.err, ERR_FA_WAIT + 7, &bar->beat);
                s_ph ^= 1;
                tc_fence_after();
                float s[128];
#pragma unroll
                for (int c = 0; c < 4; c++) tm_ld32(ts + 32 * c, s + 32 * c);
                tc_wait_ld();
                // rows that are no query's (and the next sequence's) are not masked: nobody reads them
                const int lim = valid ? vis - (w.kv0 + i) * kFaTile : kFaTile;
                if (!(p.scale_log2 > 0.0f)) {
                    const float turn = p.scale_log2 < 0.0f ? -1.0f : 0.0f;
#pragma unroll
                    for (int c = 0; c < 128; c++) s[c] *= turn;
                }
                if (__any_sync(0xffffffffu, lim < kFaTile || !there)) {
                    if (!__all_sync(0xffffffffu, there)) {
                        ok = false;
                        break;
                    }
#pragma unroll
                    for (int c = 0; c < 128; c++) s[c] = c < lim ? s[c] : -INFINITY;
                }
                float mx[4] = {max3(s[0], s[4], s[8]), max3(s[1], s[5], s[9]), max3(s[2], s[6], s[10]), max3(s[3], s[7], s[11])};
#pragma unroll
                for (int c = 12; c < 124; c += 8)
#pragma unroll
                    for (int e = 0; e < 4; e++) mx[e] = max3(mx[e], s[c + e], s[c + 4 + e]);
                const float mn = max3(max3(mx[0], mx[1], max3(s[124], s[125], s[126])), max3(mx[2], mx[3], s[127]), m);
                if (i == 0) {
                    m = mn;
                } else {
                    const bool grow = (mn - m) * scale > 8.0f;
                    if (__any_sync(0xffffffffu, grow)) {
                        // these scores came after the product before them: the output is at rest
                        const float f = grow ? exp2_fast((m - mn) * scale) : 1.0f;
                        m = grow ? mn : m;
                        l *= f;
#pragma unroll
                        for (int c = 0; c < D / 16; c++) {
                            float o[16];
                            tm_ld16(to + 16 * c, o);
                            tc_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; e++) o[e] *= f;
                            tm_st16(to + 16 * c, reinterpret_cast<const uint32_t*>(o));
                        }
                    }
                }
                const float base = m == -INFINITY ? 0.0f : fmaf(m, scale, kFaDown);
                float2 ls = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const float2 x = ffma2(make_float2(s[32 * c + 2 * e], s[32 * c + 2 * e + 1]), make_float2(scale, scale),
                                               make_float2(-base, -base));
                        // every eighth pair on the FMA units (the same prompts: none 584-600 us, an eighth 569, a quarter
                        // 610-630); not beside the conversion warps, which need those units (609 us none, 636 an eighth)
                        const float2 y = !F8 && e % 8 == 0 ? exp2_fma(x) : make_float2(exp2_fast(x.x), exp2_fast(x.y));
                        ls = ffma2(y, make_float2(1.0f, 1.0f), ls);
                        const __nv_bfloat162 v = __floats2bfloat162_rn(y.x, y.y);  // weights in 8 bits' mantissa, as the tensor cores take bf16
                        pk[e] = *reinterpret_cast<const uint32_t*>(&v);
                    }
                    tm_st16(ts + 16 * c, pk);
                    if ((c + 1) % (4 / kFaParts) == 0) {  // the product takes these positions while the next weights are made
                        tm_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&bar->p_ready[h][(c + 1) / (4 / kFaParts) - 1]);
                    }
                }
                l += ls.x + ls.y;
            }
            if (!ok) break;
            // ---- the row's output ----
            const bool any = w.nh[h] > 0;
            if (any) {
                if (!fa_wait(&bar->o_full[h], o_ph, p.err, ERR_FA_WAIT + 8, &bar->beat)) {
                    ok = false;
                    break;
                }
                o_ph ^= 1;
                tc_fence_after();
            }
            const bool wide = ((reinterpret_cast<uintptr_t>(p.out) | (static_cast<uintptr_t>(p.out_stride) * 2)) & 31u) == 0;
            const float inv = w.slot >= 0 ? 1.0f : vis > 0 ? 1.0f / l : 0.0f;
            const int head = w.kvh * p.G + head_of;
            uint16_t* out = p.out + static_cast<int64_t>(w.s.q0 + token) * p.out_stride + static_cast<int64_t>(head) * D;
            float* line = ws.part + ((static_cast<int64_t>(max(w.slot, 0)) * p.Hkv + w.kvh) * kFaRows + h * kFaTile + row) * fa_line(D);
            bool odd = !(l <= 3.4e38f);
#pragma unroll
            for (int c = 0; c < D / 32; c++) {
                float o[32];
                if (any) {
                    tm_ld32(to + 32 * c, o);
                    tc_wait_ld();
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = 0.0f;
                }
                float bad = 0.0f;
#pragma unroll
                for (int e = 0; e < 32; e++) {
                    o[e] = vis > 0 ? o[e] * inv : 0.0f;
                    bad = fmaf(o[e], 0.0f, bad);
                }
                odd |= bad != 0.0f;  // NaN unless every value is finite
                if (!valid) continue;
                if (w.slot < 0) {
#pragma unroll
                    for (int e = 0; e < 32; e += 16) {
                        uint32_t v[8];
#pragma unroll
                        for (int k = 0; k < 8; k++) {
                            const __nv_bfloat162 b2 = __floats2bfloat162_rn(o[e + 2 * k], o[e + 2 * k + 1]);
                            v[k] = *reinterpret_cast<const uint32_t*>(&b2);
                        }
                        if (wide) {
                            st_global_v8(out + 32 * c + e, v);
                        } else {
                            *reinterpret_cast<uint4*>(out + 32 * c + e) = make_uint4(v[0], v[1], v[2], v[3]);
                            *reinterpret_cast<uint4*>(out + 32 * c + e + 8) = make_uint4(v[4], v[5], v[6], v[7]);
                        }
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e += 8)
                        st_global_v8(line + 32 * c + e, *reinterpret_cast<const uint32_t(*)[8]>(&o[e]));
                }
            }
            if (w.slot >= 0 && valid) *reinterpret_cast<float2*>(line + D) = make_float2(m == -INFINITY ? m : m * scale, l);
            const unsigned again = __ballot_sync(0xffffffffu, valid && odd);
            if (again)
                fa_redo<KIND, D>(p, w.b, w.base, w.kvh, w.kv0 * kFaTile, min(w.s.len, (w.kv0 + w.nh[h]) * kFaTile), again, w.s.q0 + token, head, vis,
                                 w.slot < 0 ? nullptr : line, lane, &bar->beat);
            tc_fence_before();
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Geo::REST_REGS));
        if (warp == kFaSoft + 1) {
            // ---- loader (of the codes' slots when they are to be converted) ----
            Ring<F8 ? 2 : ST> r;
            uint64_t* const full_bar = F8 ? bar->raw_full : bar->kv_full;
            uint64_t* const empty_bar = F8 ? bar->raw_empty : bar->kv_empty;
            unsigned q_phase = 0, q_loads[2] = {0, 0};
            bool ok = true;
            const int32_t* table = nullptr;
            int ids_of = -1, ids = 0, ids_next = 0;
            const int per_tile = kFaTile >> p.kv.page_log2;  // pages of a tile
            auto lookup = [&](int tile) {
                int id = 0;
                const int at = tile * per_tile + lane;
                if (lane < per_tile && at < p.kv.max_pages) id = __ldcg(table + at);
                return id;
            };
            // Planned before: the next unit's record is fetched while the current one is loaded.
            auto listed = [&](int u) {  // lanes 0 and 1: its two halves
                return lane < 2 && u / p.Hkv < ws.max_units ? __ldcg(reinterpret_cast<const int4*>(ws.units + u / p.Hkv) + lane) : make_int4(0, 0, 0, 0);
            };
            FaTiles own;
            if (ws.direct)
                own = fa_plan_tiles(p.q_start, p.kv_len, p.B, p.T, p.kv_max, p.max_q, p.Hkv, ws.sms, tq, lane, ws.splits, ws.head,
                                    blockIdx.x == 0 ? p.err : nullptr);
            auto record = [&](int u) { return ws.direct ? own.unit(u / p.Hkv, lane) : listed(u); };
            int next = blockIdx.x;
            int4 rec = record(next);
            const int units = (ws.direct ? own.units : __ldcg(&ws.head->units)) * p.Hkv;
            while (ok) {
                const int u = next;
                if (!fa_wait(&bar->u_empty[feed.i], feed.phase ^ 1, p.err, ERR_FA_WAIT + 13, &bar->beat)) break;
                if (lane < 2) reinterpret_cast<int4*>(&bar->unit[feed.i])[lane] = rec;
                if (lane == 0) bar->kvh[feed.i] = u < units ? u % p.Hkv : -1;
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar->u_full[feed.i]);
                const FaWork w = fa_work(p, bar->unit[feed.i], u % p.Hkv, tq);
                feed.next();
                if (u >= units) break;
                if (lane == 0) next = ws.direct ? u + gridDim.x : gridDim.x + atomicAdd(&ws.head->next, 1);
                next = __shfl_sync(0xffffffffu, next, 0);
                rec = record(next);
                if (w.keys == 0) continue;
                if constexpr (KIND != KV_ROWS) {
                    table = p.kv.table + static_cast<int64_t>(w.b) * p.kv.table_stride;
                    ids_of = w.kv0;
                    ids = lookup(ids_of);
                    ids_next = w.keys > 1 ? lookup(ids_of + 1) : 0;
                }
                auto load = [&](bool value, int tile, int page_ids) {
                    if (!ok || !fa_wait(&empty_bar[r.i], r.phase ^ 1, p.err, ERR_FA_WAIT + 1, &bar->beat)) {
                        ok = false;
                        return;
                    }
                    uint8_t* dst = smem + (F8 ? Geo::RAW_OFF + r.i * Geo::CODES : Geo::KV_OFF + r.i * Geo::TILE);
                    uint64_t* full = &full_bar[r.i];
                    const CUtensorMap* map = value ? &vmap : &kmap;
                    if constexpr (KIND == KV_ROWS) {
                        if (lane == 0) {
                            mbar_arrive_expect_tx(full, Geo::TILE);
#pragma unroll
                            for (int c = 0; c < CH; c++)
                                tma_load_3d(dst + c * Geo::HALF, map, c * 64, w.kvh, w.base + tile * kFaTile, full);
                        }
                    } else {
                        const int page = 1 << p.kv.page_log2;
                        const int have = min(per_tile, (w.s.len - tile * kFaTile + page - 1) >> p.kv.page_log2);
                        const bool mine = lane < have;
                        const bool good = mine && page_ids >= 0 && page_ids < p.kv.num_pages;
                        if (mine && !good && !value) record_error(p.err, ERR_KV_TABLE);
                        const int exps = F8 ? __popc(__ballot_sync(0xffffffffu, good)) * page : 0;
                        if (lane == 0) mbar_arrive_expect_tx(full, have * page * D * (F8 ? 1 : 2) + exps);
                        __syncwarp();
                        if (mine) {
                            const int id = good ? page_ids : p.kv.num_pages;  // outside the map: zeros
                            if constexpr (F8) {
                                tma_load_4d(dst + lane * page * D, map, 0, 0, w.kvh, id, full);
                                if (good)
                                    bulk_g2s_plain(smem + Geo::EXP_OFF + r.i * kFaTile + lane * page,
                                                   (value ? p.kv.ve : p.kv.ke) + id * p.kv.exp_stride + (static_cast<int64_t>(w.kvh) << p.kv.page_log2),
                                                   page, full);
                            } else {
#pragma unroll
                                for (int c = 0; c < CH; c++)
                                    tma_load_4d(dst + c * Geo::HALF + lane * page * 128, map, c * 64, 0, w.kvh, id, full);
                            }
                        }
                    }
                    r.next();
                };
                load(false, w.kv0, ids);
                // the queries, once the previous unit's last scores are multiplied
                if (ok && !fa_wait(&bar->q_empty, q_phase ^ 1, p.err, ERR_FA_WAIT + 2, &bar->beat)) ok = false;
                q_phase ^= 1;
                if (!ok) break;
#pragma unroll
                for (int h = 0; h < 2; h++) q_loads[h] += w.nh[h] > 0;
                if (lane == 0) {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        if (w.nh[h] == 0) continue;
                        mbar_arrive_expect_tx(&bar->q_full[h], tq * p.G * D * 2);
#pragma unroll
                        for (int c = 0; c < CH; c++)
                            tma_load_3d(smem + Geo::Q_OFF + h * Geo::TILE + c * Geo::HALF, &qmap, c * 64, w.kvh * p.G,
                                        w.s.q0 + w.i0 + h * tq, &bar->q_full[h]);
                    }
                }
                __syncwarp();
                for (int i = 0; i < w.keys && ok; i++) {
                    const int cur = ids;
                    if (i + 1 < w.keys) {
                        ids = ids_next;
                        if (KIND != KV_ROWS && i + 2 < w.keys) ids_next = lookup(w.kv0 + i + 2);
                        load(false, w.kv0 + i + 1, ids);
                    }
                    load(true, w.kv0 + i, cur);
                }
            }
            // the last loads of every slot have landed before the CTA ends, whoever still waited for them: nothing may arrive
            // in its shared memory later (a slot never loaded counts as landed)
            for (int i = 0; i < (F8 ? 2 : ST); i++) {
                fa_drain(&full_bar[r.i], r.phase ^ 1, p.err, ERR_FA_WAIT + 3);
                r.next();
            }
#pragma unroll
            for (int h = 0; h < 2; h++)
                if (q_loads[h]) fa_drain(&bar->q_full[h], (q_loads[h] - 1) & 1, p.err, ERR_FA_WAIT + 3);
        } else if (F8 && warp >= kFaSoft + 4) {
            // ---- conversion: codes times their row's power of two, exact in bf16, into the swizzled tile ----
            Ring<2> rr;
            Ring<ST> r;
            bool ok = true;
            constexpr int RC = D / 16;  // 16-code chunks of a row
            const int ct = tid - (kFaSoft + 4) * 32;
            auto convert = [&](int left) {
                if (!ok) return;
                const bool raw = fa_wait_lane(&bar->raw_full[rr.i], rr.phase, p.err, ERR_FA_WAIT + 9, &bar->beat);
                if (!__all_sync(0xffffffffu, fa_wait_lane(&bar->kv_empty[r.i], r.phase ^ 1, p.err, ERR_FA_WAIT + 10, &bar->beat) && raw)) {
                    ok = false;
                    return;
                }
                const uint8_t* codes = smem + Geo::RAW_OFF + rr.i * Geo::CODES;
                const uint8_t* exps = smem + Geo::EXP_OFF + rr.i * kFaTile;
                uint8_t* dst = smem + Geo::KV_OFF + r.i * Geo::TILE;
#pragma unroll 2
                for (int o = ct; o < kFaTile * RC; o += 128) {
                    const int row = o / RC, c = o % RC;
                    const uint4 w = *reinterpret_cast<const uint4*>(codes + o * 16);
                    // a byte of 255 (a slot that was never written, or a page outside the pool) must not make NaN of zeros
                    const float sc = exp_byte(min(static_cast<unsigned>(exps[row]), 254u));
                    const unsigned u[4] = {w.x, w.y, w.z, w.w};
                    uint32_t v[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float2 f = e4m3x2_to_float2(static_cast<unsigned short>(u[i / 2] >> (16 * (i & 1))));
                        const float2 g = fmul2(f, make_float2(sc, sc));
                        const __nv_bfloat162 b2 = __floats2bfloat162_rn(g.x, g.y);
                        v[i] = *reinterpret_cast<const uint32_t*>(&b2);
                    }
                    if (row >= left) {  // behind the last position: anything may be there, and 0 * NaN is NaN
#pragma unroll
                        for (int i = 0; i < 8; i++) v[i] = 0u;
                    }
                    // chunks 2 (c % 4) and + 1 of the row's 64-column half; the upper half writes them in the other order, so
                    // that eight lanes of a row meet eight bank groups
                    uint8_t* at = dst + (c / 4) * Geo::HALF + row * 128;
                    const int first = c / 4, k0 = 2 * (c % 4) + first, k1 = 2 * (c % 4) + 1 - first;
                    const uint4 lo = make_uint4(v[0], v[1], v[2], v[3]), hi = make_uint4(v[4], v[5], v[6], v[7]);
                    *reinterpret_cast<uint4*>(at + ((k0 ^ (row & 7)) << 4)) = first ? hi : lo;
                    *reinterpret_cast<uint4*>(at + ((k1 ^ (row & 7)) << 4)) = first ? lo : hi;
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&bar->kv_full[r.i]);
                    mbar_arrive(&bar->raw_empty[rr.i]);
                }
                rr.next();
                r.next();
            };
            for (FaWork w; ok && take(w);) {
                if (w.keys == 0) continue;
                convert(w.s.len - w.kv0 * kFaTile);
                for (int i = 0; i < w.keys && ok; i++) {
                    const int left = w.s.len - (w.kv0 + i) * kFaTile;
                    if (i + 1 < w.keys) convert(left - kFaTile);
                    convert(left);
                }
            }
        } else if (warp == kFaSoft) {
            // ---- the issuing warp ----
            Ring<ST> r;
            unsigned q_ph[2] = {0, 0}, p_ph[2] = {0, 0};
            bool ok = true;
            constexpr uint32_t id_s = fa_idesc(kFaTile, false), id_o = fa_idesc(D, true);
            bool gone = false;  // this lane gave up
            auto wait = [&](uint64_t* b, unsigned ph, int role) { gone |= !fa_wait_lane(b, ph, p.err, ERR_FA_WAIT + role, &bar->beat); };
            const uint32_t q_lo = uniform(static_cast<uint32_t>(tc_smem_desc(smem_addr(smem + Geo::Q_OFF))));
            const uint32_t k_lo = uniform(static_cast<uint32_t>(tc_smem_desc(smem_addr(smem + Geo::KV_OFF))));
            const uint32_t v_lo = uniform(static_cast<uint32_t>(fa_desc_mn(smem_addr(smem + Geo::KV_OFF), Geo::HALF)));
            constexpr uint32_t k_hi = static_cast<uint32_t>(tc_smem_desc(0) >> 32), v_hi = static_cast<uint32_t>(fa_desc_mn(0, 0) >> 32);
            const uint32_t tm = uniform(tmem);
            auto scores = [&](int h, int stage) {
                tc_fence_after();
                const uint32_t q = q_lo + h * (Geo::TILE >> 4), k = uniform(k_lo + stage * (Geo::TILE >> 4));
                if (elect_one()) {
#pragma unroll
                    for (int i = 0; i < D / 16; i++) {
                        const uint32_t off = ((i / 4) * Geo::HALF + (i % 4) * 32) >> 4;
                        fa_mma_ss(tm + h * 128, q + off, k + off, k_hi, id_s, i > 0);
                    }
                    tc_commit(&bar->s_full[h]);
                }
                __syncwarp();
            };
            // the product with a part of the tile's positions
            auto outputs = [&](int h, int stage, int part, bool first, bool final) {
                tc_fence_after();
                constexpr int N = kFaTile / 16 / kFaParts;
                const uint32_t v = uniform(v_lo + stage * (Geo::TILE >> 4) + part * (N * 2048 >> 4));
                const uint32_t a = uniform(tm + h * 128 + part * N * 8);
                const int more = uniform(part > 0 || !first);
                if (elect_one()) {
#pragma unroll
                    for (int i = 0; i < N; i++)
                        fa_mma_ts(tm + 256 + h * 128, a + i * 8, v + i * (2048 >> 4), v_hi, id_o, i > 0 ? 1 : more);
                    if (final) tc_commit(&bar->o_full[h]);
                }
                __syncwarp();
            };
            auto release = [&](uint64_t* b) {
                if (elect_one()) tc_commit(b);
                __syncwarp();
            };
            for (FaWork w; ok && take(w);) {
                if (w.keys == 0) continue;
                wait(&bar->kv_full[r.i], r.phase, 4);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if (w.nh[h] == 0) continue;
                    wait(&bar->q_full[h], q_ph[h], 5);
                    q_ph[h] ^= 1;
                    scores(h, r.i);
                }
                release(&bar->kv_empty[r.i]);
                r.next();
                if (w.keys == 1) release(&bar->q_empty);
                for (int i = 0; i < w.keys && ok; i++) {
                    const bool more = i + 1 < w.keys;
                    int k_stage = 0;
                    if (more) {
                        k_stage = r.i;
                        wait(&bar->kv_full[r.i], r.phase, 4);
                        r.next();
                    }
                    const int v_stage = r.i;
                    wait(&bar->kv_full[r.i], r.phase, 4);
                    r.next();
                    const int left = w.s.len - (w.kv0 + i) * kFaTile;  // positions of the tile
                    if (!F8 && left < kFaTile) {
                        // rows behind the last position: anything may be there, and 0 * NaN is NaN
                        uint8_t* v = smem + Geo::KV_OFF + v_stage * Geo::TILE;
                        for (int o = left * 8 + lane; o < kFaTile * 8; o += 32)
#pragma unroll
                            for (int c = 0; c < CH; c++) *reinterpret_cast<uint4*>(v + c * Geo::HALF + o * 16) = make_uint4(0u, 0u, 0u, 0u);
                        fence_async_smem();
                        __syncwarp();
                    }
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        if (i >= w.nh[h]) continue;
                        for (int part = 0; part < kFaParts; part++) {
                            wait(&bar->p_ready[h][part], p_ph[h], 6);
                            outputs(h, v_stage, part, i == 0, part + 1 == kFaParts && i + 1 == w.nh[h]);
                        }
                        p_ph[h] ^= 1;
                        if (i + 1 < w.nh[h]) scores(h, k_stage);
                    }
                    ok = !__any_sync(0xffffffffu, gone);
                    if (!ok) break;
                    release(&bar->kv_empty[v_stage]);
                    if (more) release(&bar->kv_empty[k_stage]);
                    if (i + 2 == w.keys) release(&bar->q_empty);
                }
            }
            // every product has read its operands before the CTA ends, also where the softmax gave up on one
            release(&bar->done);
            fa_drain(&bar->done, 0, p.err, ERR_FA_WAIT + 14);
        }
    }
    __syncthreads();
    if (warp == kFaSoft) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// Rows whose positions were split: parts joined in order, one warp a row.
template <int KIND, int D>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ PattnParams p, const __grid_constant__ FaWs ws) {
    constexpr int E = D / 32;
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int tq = fa_tokens(p.G);
    // a split tile's record and how many there are, read at once (the list is longer than the tiles can be)
    int most = ws.max_slots * p.Hkv * kFaRows;  // 512 rows an SM, or two slots
    const int splits = __ldcg(&ws.head->splits);
    for (int i = blockIdx.x * 8 + (threadIdx.x >> 5); i < most; i += gridDim.x * 8) {
        const int r = i % kFaRows, tile = i / kFaRows, of = tile / p.Hkv, kvh = tile - of * p.Hkv;
        const int4* at = reinterpret_cast<const int4*>(ws.splits + of);
        const int4 sa = __ldcg(at), sb = __ldcg(at + 1);  // q0, n, len, i0; b, slot, parts
        most = splits * p.Hkv * kFaRows;
        if (i >= most) break;
        const int hr = r % kFaTile;
        const int token = sa.w + (r / kFaTile) * tq + hr / p.G, head = kvh * p.G + hr % p.G;
        if (hr / p.G >= tq || token >= sa.y) continue;
        const int vis = max(0, min(sa.z, sa.z - sa.y + token + 1));
        const float* base = ws.part + ((static_cast<int64_t>(sb.y) * p.Hkv + kvh) * kFaRows + r) * fa_line(D);
        const int64_t step = static_cast<int64_t>(p.Hkv) * kFaRows * fa_line(D);
        // sixteen parts' loads under way at once
        float M = -INFINITY, a[E] = {}, l = 0.0f;
        for (int j0 = 0; j0 < sb.z; j0 += 16) {
            float2 ml[16], v[16][E / 2];
            float mn = M;
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const bool in = j0 + j < sb.z;
                const float* pr = base + (j0 + j) * step;
                ml[j] = in ? __ldcg(reinterpret_cast<const float2*>(pr + D)) : make_float2(-INFINITY, 0.0f);
#pragma unroll
                for (int e = 0; e < E / 2; e++)
                    v[j][e] = in ? __ldcg(reinterpret_cast<const float2*>(pr + lane * E + 2 * e)) : make_float2(0.0f, 0.0f);
            }
#pragma unroll
            for (int j = 0; j < 16; j++) mn = fmaxf(mn, ml[j].x);
            const float b0 = mn == -INFINITY ? 0.0f : mn, c = exp2_fast(M - b0);
            M = mn;
            l *= c;
#pragma unroll
            for (int e = 0; e < E; e++) a[e] *= c;
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const float f = exp2_fast(ml[j].x - b0);
                l = fmaf(f, ml[j].y, l);
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    a[e] = fmaf(f, v[j][e / 2].x, a[e]);
                    a[e + 1] = fmaf(f, v[j][e / 2].y, a[e + 1]);
                }
            }
        }
        const float inv = vis > 0 ? 1.0f / l : 0.0f;
        uint16_t* o = p.out + static_cast<int64_t>(sa.x + token) * p.out_stride + static_cast<int64_t>(head) * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            const __nv_bfloat162 b2 = __floats2bfloat162_rn(a[e] * inv, a[e + 1] * inv);
            *reinterpret_cast<__nv_bfloat162*>(o + e) = b2;
        }
    }
}

}  // namespace oomb
