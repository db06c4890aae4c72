// pdecode.cuh - attention of a few query rows per kv head over a paged cache: decode
// steps and short drafts, up to 16 rows (new tokens x query heads of a kv head).
//
// Bound: HBM; every key and value byte is read once and used for all rows at once.  The
// 16 rows are one M = 16 tile of the warp-level matrix instructions (mma.m16n8k16); the
// 128-row tiles of the 5th-generation tensor cores would leave 7/8 of their rows empty
// and pass every key through tensor memory for nothing: at the measured HBM rate an SM gets
// 16 positions (8 KB in bf16) every ~185 ns and needs 32 such instructions for them.
//
// Work split: the batch's positions are cut into blocks of 128 (per sequence and kv head)
// and the blocks, laid end to end, evenly over the CTAs (one per SM), whatever the lengths;
// a (sequence, kv head) spread over several CTAs is joined by the last of them
// to finish, in order, so a call's bits do not depend on timing.  Within a CTA each warp
// takes every eighth group of 16 positions with a running maximum and sum of its own.
//
// Loads: each warp keeps a ring of groups in flight with cp.async, and every byte is
// fetched by the one lane that will use it, so the ring needs no barrier and no
// transpose.  That works because both products may order their inner index freely:
//  - scores: lane (g = lane / 4, t = lane % 4) is the B fragment's column g (a position) and
//    four inner indices a step; it takes 16-byte chunks of the rows of positions g and
//    8 + g, and the query fragment is laid out with the same order of dimensions;
//  - values: the lane holds positions 2t, 2t + 1, 2t + 8, 2t + 9 (the inner index) and column g,
//    and a column may stand for any dimension: it takes whole chunks of those four rows
//    and pairs two positions' values with byte permutes.
// e4m3 codes become f16 exactly (one conversion a pair); queries are then f16 too, each
// row scaled by a power of two so that its largest value lies in [2^13, 2^14): their eight
// bits stay exact down to 2^-28 of it.  Keys' exponents multiply the scores; values'
// join the weights as w = p 2^(e - X), X the largest exponent met so far, so w <= 1 and fits f16.
#pragma once

#include "pattn.cuh"

namespace oomb {

constexpr int kDecWarps = 8;
constexpr int kDecThreads = kDecWarps * 32;
constexpr int kDecBlock = 128;   // positions of a work block: one group of 16 a warp
constexpr int kDecRows = 16;
constexpr int kDecRingBytes = 192 * 1024;

template <int KIND, int D>
struct DecodeGeo {
    static constexpr bool F8 = KIND == KV_E4M3;
    static constexpr int ROW = F8 ? D : 2 * D;                 // bytes of a position's row
    static constexpr int KC = ROW / 64;                        // 16-byte chunks of a key row a lane takes
    static constexpr int VB = ROW / 8 < 16 ? ROW / 8 : 16;     // bytes of a value chunk (8 lanes a row)
    static constexpr int VC = ROW / 8 / VB;                    // value chunks of a row a lane takes
    static constexpr int STAGE = 16 * ROW * 2;                 // keys and values of a group
    static constexpr int STAGES = kDecRingBytes / (kDecWarps * STAGE) < 8 ? kDecRingBytes / (kDecWarps * STAGE) : 8;
    static constexpr int PAD = D + 4;                          // floats of a merge row
    static constexpr size_t smem = static_cast<size_t>(kDecWarps) * STAGE * STAGES + kDecWarps * STAGES * 32;
    static_assert(static_cast<size_t>(kDecWarps) * kDecRows * PAD * 4 <= static_cast<size_t>(kDecWarps) * STAGE * STAGES,
                  "the merge rows reuse the ring");
};

struct DecodeWs {
    unsigned* counters;  // [grid] arrivals, zero between launches
    float* part;         // [2 * grid][rows][D + 4]: acc, m, l
    int rows;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, unsigned bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp8(uint32_t dst, const void* src, unsigned bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, unsigned bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <bool F16>
__device__ __forceinline__ void mma16816(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                         unsigned b1) {
    if constexpr (F16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Two e4m3 codes (low half of w) as two f16.
__device__ __forceinline__ unsigned f16x2_of(unsigned w) {
    unsigned r;
    asm("{\n .reg .b16 l;\n cvt.u16.u32 l, %1;\n cvt.rn.f16x2.e4m3x2 %0, l;\n}" : "=r"(r) : "r"(w));
    return r;
}
__device__ __forceinline__ unsigned pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&h);
}

// First block of CTA c of n over `total` blocks, and the CTA that owns a block.
__device__ __forceinline__ int64_t dec_lo(int64_t total, int c, int n) { return total * c / n; }
__device__ __forceinline__ int dec_owner(int64_t total, int64_t block, int n) {
    int c = static_cast<int>(block * n / total);
    while (c + 1 < n && dec_lo(total, c + 1, n) <= block) c++;
    while (c > 0 && dec_lo(total, c, n) > block) c--;
    return c;
}

template <int KIND, int D>
__global__ void __launch_bounds__(kDecThreads, 1) decode_rows_kernel(const __grid_constant__ PattnParams p, const DecodeWs ws) {
    using Geo = DecodeGeo<KIND, D>;
    constexpr bool F8 = Geo::F8;
    constexpr int KC = Geo::KC, VC = Geo::VC, VB = Geo::VB, STAGES = Geo::STAGES, PAD = Geo::PAD;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int64_t scan_sum[kDecWarps];
    __shared__ int64_t start_prefix;
    __shared__ int start_b;
    __shared__ float mls[kDecWarps][kDecRows][2];
    __shared__ bool last;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    uint8_t* ring = smem + warp * Geo::STAGE * STAGES;
    const uint32_t ring_s = smem_addr(ring);
    uint8_t* exps = smem + static_cast<size_t>(kDecWarps) * Geo::STAGE * STAGES + warp * STAGES * 32;
    const uint32_t exps_s = smem_addr(exps);

    pdl_wait();
    pdl_launch_dependents();

    // ---- this CTA's blocks of the batch ----
    auto blocks_of = [&](int b) {
        if (b >= p.B) return 0;
        const Seq s = read_seq(p.q_start, p.kv_len, b, p.T, p.kv_max, p.err);
        if (s.n > p.max_q) record_error(p.err, ERR_KV_SEQ);
        if (s.n == 0 || s.n > p.max_q) return 0;
        return max(1, (s.len + kDecBlock - 1) / kDecBlock);  // a sequence without positions still gets its zeros
    };
    int64_t total = 0;
    int mine = 0;
    for (int b0 = 0; b0 < p.B; b0 += kDecThreads) {
        mine = blocks_of(b0 + tid);
        int v = mine;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == 0) scan_sum[warp] = v;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kDecWarps; w++) total += scan_sum[w];
        __syncthreads();
    }
    const int64_t W = total * p.Hkv;
    const int S = static_cast<int>(W < static_cast<int64_t>(gridDim.x) ? W : static_cast<int64_t>(gridDim.x));
    const int cta = blockIdx.x;
    if (cta >= S) return;
    int64_t lo = dec_lo(W, cta, S);
    const int64_t hi = dec_lo(W, cta + 1, S);
    int64_t prefix = 0;
    for (int b0 = 0; b0 < p.B; b0 += kDecThreads) {
        if (p.B > kDecThreads) mine = blocks_of(b0 + tid);
        int inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += u;
        }
        if (lane == 31) scan_sum[warp] = inc;
        __syncthreads();
        int64_t before = prefix;
        for (int w = 0; w < warp; w++) before += scan_sum[w];
        const int64_t end = before + inc;
        if (mine > 0 && (end - mine) * p.Hkv <= lo && lo < end * p.Hkv) {
            start_b = b0 + tid;
            start_prefix = end - mine;
        }
#pragma unroll
        for (int w = 0; w < kDecWarps; w++) prefix += scan_sum[w];
        __syncthreads();
    }
    int b = start_b;
    int64_t b_first = start_prefix * p.Hkv;  // first block of sequence b

    // ---- segments: the CTA's blocks of one (sequence, kv head) at a time ----
    while (lo < hi) {
        Seq sq = read_seq(p.q_start, p.kv_len, b, p.T, p.kv_max, nullptr);
        const int nb = sq.n == 0 || sq.n > p.max_q ? 0 : max(1, (sq.len + kDecBlock - 1) / kDecBlock);
        if (lo >= b_first + static_cast<int64_t>(nb) * p.Hkv) {
            b_first += static_cast<int64_t>(nb) * p.Hkv;
            b++;
            continue;
        }
        const int kvh = static_cast<int>((lo - b_first) / nb);
        const int64_t pair_first = b_first + static_cast<int64_t>(kvh) * nb, pair_end = pair_first + nb;
        const int64_t seg_end = pair_end < hi ? pair_end : hi;
        const int tok0 = static_cast<int>(lo - pair_first) * kDecBlock;
        const int tok1 = min(sq.len, static_cast<int>(seg_end - pair_first) * kDecBlock);
        const int rows = sq.n * p.G;
        const int groups = tok1 > tok0 ? (tok1 - tok0 + 15) / 16 : 0;
        const int count = groups > warp ? (groups - warp + kDecWarps - 1) / kDecWarps : 0;  // this warp's groups

        // the queries' fragments: rows g and 8 + g
        unsigned qa[D / 16][4];
        float row_scale[2];
        int vis[2];
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const int r = g + 8 * half;
            const bool ok = r < rows;
            const int token = ok ? r / p.G : 0;
            vis[half] = ok ? max(0, min(sq.len, sq.len - sq.n + token + 1)) : 0;
            const uint16_t* qp = p.q + static_cast<int64_t>(sq.q0 + token) * p.q_stride + static_cast<int64_t>(kvh * p.G + (ok ? r - token * p.G : 0)) * D;
            row_scale[half] = p.scale_log2;
            if constexpr (!F8) {
#pragma unroll
                for (int c = 0; c < D / 32; c++) {
                    const uint4 w = ok ? __ldcg(reinterpret_cast<const uint4*>(qp + c * 32 + t * 8)) : make_uint4(0u, 0u, 0u, 0u);
                    qa[2 * c][half] = w.x;
                    qa[2 * c][half + 2] = w.y;
                    qa[2 * c + 1][half] = w.z;
                    qa[2 * c + 1][half + 2] = w.w;
                }
            } else {
                unsigned u[D / 64][8];
                float amax = 0.0f;
#pragma unroll
                for (int c = 0; c < D / 64; c++) {
                    const uint4* src = reinterpret_cast<const uint4*>(qp + c * 64 + t * 16);
                    const uint4 w0 = ok ? __ldcg(src) : make_uint4(0u, 0u, 0u, 0u), w1 = ok ? __ldcg(src + 1) : make_uint4(0u, 0u, 0u, 0u);
                    u[c][0] = w0.x, u[c][1] = w0.y, u[c][2] = w0.z, u[c][3] = w0.w;
                    u[c][4] = w1.x, u[c][5] = w1.y, u[c][6] = w1.z, u[c][7] = w1.w;
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(u[c][i] << 16)), fabsf(__uint_as_float(u[c][i] & 0xffff0000u))));
                }
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                const int ex = max(-100, min(100, static_cast<int>(__float_as_uint(amax) >> 23) - 127 - 13));
                const float up = __int_as_float((127 - ex) << 23);
                row_scale[half] = p.scale_log2 * __int_as_float((127 + ex) << 23);
#pragma unroll
                for (int c = 0; c < D / 64; c++)
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        // element pair i of the chunk: step c * 4 + i / 2, its first or second inner half
                        qa[c * 4 + i / 2][half + 2 * (i & 1)] =
                            pack_f16(__uint_as_float(u[c][i] << 16) * up, __uint_as_float(u[c][i] & 0xffff0000u) * up);
                    }
            }
        }
        const int vis_least = max(0, min(sq.len, sq.len - sq.n + 1));

        // ---- the ring of groups ----
        const int32_t* table = p.kv.table + static_cast<int64_t>(b) * p.kv.table_stride;
        const int page_mask = (1 << p.kv.page_log2) - 1;
        int ids = 0, ids_base = -32;  // lane l holds the page of the warp's group ids_base + l
        auto issue = [&](int i) {
            if (i < count) {
                if (i >= ids_base + 32) {
                    ids_base += 32;
                    const int gi = ids_base + lane;
                    ids = gi < count ? __ldcg(table + ((tok0 + (warp + gi * kDecWarps) * 16) >> p.kv.page_log2)) : 0;
                    if (ids < 0 || ids >= p.kv.num_pages) {
                        record_error(p.err, ERR_KV_TABLE);
                        ids = -1;
                    }
                }
                const int page = __shfl_sync(0xffffffffu, ids, i - ids_base);
                const int tok = tok0 + (warp + i * kDecWarps) * 16;
                const int have = page < 0 ? 0 : tok1 - tok;  // positions of the group present
                const int64_t row0 = max(page, 0) * p.kv.page_stride + ((static_cast<int64_t>(kvh) << p.kv.page_log2) + (tok & page_mask)) * D;
                const int es = F8 ? 1 : 2;
                const uint8_t* kb = p.kv.k + row0 * es;
                const uint8_t* vb = p.kv.v + row0 * es;
                const uint32_t dst = ring_s + (i % STAGES) * Geo::STAGE;
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int c = 0; c < KC; c++) {
                        const int pos = 8 * j + g;
                        cp16(dst + (j * KC + c) * 512 + lane * 16, kb + pos * Geo::ROW + c * 64 + t * 16, pos < have ? 16u : 0u);
                    }
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int c = 0; c < VC; c++) {
                        const int pos = 2 * t + (j & 1) + 8 * (j >> 1);
                        const uint32_t d = dst + 16 * Geo::ROW + (j * VC + c) * 32 * VB + lane * VB;
                        const uint8_t* s = vb + pos * Geo::ROW + c * 8 * VB + g * VB;
                        if constexpr (VB == 16) cp16(d, s, pos < have ? 16u : 0u);
                        else cp8(d, s, pos < have ? 8u : 0u);
                    }
                if constexpr (F8) {
                    if (lane < 8) {
                        const uint8_t* e = lane < 4 ? p.kv.ke : p.kv.ve;
                        const int64_t at = max(page, 0) * p.kv.exp_stride + (static_cast<int64_t>(kvh) << p.kv.page_log2) + (tok & page_mask);
                        cp4(exps_s + (i % STAGES) * 32 + lane * 4, e + at + (lane & 3) * 4, page < 0 ? 0u : 4u);
                    }
                }
            }
            cp_commit();
        };

        float acc[D / 8][4];
#pragma unroll
        for (int i = 0; i < D / 8; i++) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        int X = -1000;  // e4m3: the exponent that the accumulators are counted in
#pragma unroll
        for (int i = 0; i < STAGES - 1; i++) issue(i);
        for (int i = 0; i < count; i++) {
            issue(i + STAGES - 1);
            cp_wait<STAGES - 1>();
            const uint8_t* st = ring + (i % STAGES) * Geo::STAGE;
            const int tok = tok0 + (warp + i * kDecWarps) * 16;
            float s[2][4] = {};
            unsigned ke[2], ve[2];
            if constexpr (F8) {
                __syncwarp();  // the exponents were fetched by other lanes
                const uint8_t* ep = exps + (i % STAGES) * 32;
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    ke[j] = *reinterpret_cast<const uint16_t*>(ep + 8 * j + 2 * t);
                    ve[j] = *reinterpret_cast<const uint16_t*>(ep + 16 + 8 * j + 2 * t);
                    // a slot behind the last position may hold any byte: it must not set X
                    const int left = tok1 - (tok + 8 * j + 2 * t);
                    if (left < 2) ve[j] = left < 1 ? 0u : ve[j] & 0xffu;
                }
            }
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int c = 0; c < KC; c++) {
                    const uint4 w = *reinterpret_cast<const uint4*>(st + (j * KC + c) * 512 + lane * 16);
                    if constexpr (!F8) {
                        mma16816<false>(s[j], qa[2 * c][0], qa[2 * c][1], qa[2 * c][2], qa[2 * c][3], w.x, w.y);
                        mma16816<false>(s[j], qa[2 * c + 1][0], qa[2 * c + 1][1], qa[2 * c + 1][2], qa[2 * c + 1][3], w.z, w.w);
                    } else {
                        const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int q = 0; q < 4; q++)
                            mma16816<true>(s[j], qa[4 * c + q][0], qa[4 * c + q][1], qa[4 * c + q][2], qa[4 * c + q][3],
                                           f16x2_of(u[q]), f16x2_of(u[q] >> 16));
                    }
                }
            // scores in units of log2; rows g (half 0) and 8 + g (half 1), positions 8 j + 2 t + (0, 1)
            float mx[2] = {-INFINITY, -INFINITY};
            const bool masked = tok + 16 > vis_least;
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int half = e >> 1;
                    float f = row_scale[half];
                    if constexpr (F8) f *= exp_byte((ke[j] >> (8 * (e & 1))) & 0xffu);
                    float x = s[j][e] * f;
                    if (masked && tok + 8 * j + 2 * t + (e & 1) >= vis[half]) x = -INFINITY;
                    s[j][e] = x;
                    mx[half] = fmaxf(mx[half], x);
                }
#pragma unroll
            for (int half = 0; half < 2; half++) {
                mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], 1));
                mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], 2));
            }
            int xm = X;
            if constexpr (F8) {
                int e4 = max(max(static_cast<int>(ve[0] & 0xffu), static_cast<int>(ve[0] >> 8)),
                             max(static_cast<int>(ve[1] & 0xffu), static_cast<int>(ve[1] >> 8)));
                e4 = max(e4, __shfl_xor_sync(0xffffffffu, e4, 1));
                e4 = max(e4, __shfl_xor_sync(0xffffffffu, e4, 2));
                xm = max(X, e4);
            }
            if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1] || xm > X)) {
                float grow = 1.0f;
                if constexpr (F8) {
                    grow = X < -500 ? 1.0f : exp2_fast(static_cast<float>(X - xm));
                    X = xm;
                }
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const float mn = fmaxf(m[half], mx[half]);
                    const float c = m[half] == -INFINITY ? 0.0f : exp2_fast(m[half] - mn);
                    m[half] = mn;
                    l[half] *= c;
                    const float cg = c * grow;
#pragma unroll
                    for (int n = 0; n < D / 8; n++) {
                        acc[n][2 * half] *= cg;
                        acc[n][2 * half + 1] *= cg;
                    }
                }
            }
            const float base[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
            unsigned pa[4];
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    float e0 = exp2_fast(s[j][2 * half] - base[half]), e1 = exp2_fast(s[j][2 * half + 1] - base[half]);
                    l[half] += e0 + e1;
                    if constexpr (F8) {
                        // weight times 2^(e - X) <= 1; f16 keeps it to 2^-11, or to 2^-25 absolute
                        e0 *= exp2_fast(static_cast<float>(static_cast<int>(ve[j] & 0xffu) - X));
                        e1 *= exp2_fast(static_cast<float>(static_cast<int>(ve[j] >> 8) - X));
                        pa[2 * j + half] = pack_f16(e0, e1);
                    } else {
                        pa[2 * j + half] = pack_bf16(e0, e1);  // weights in 8 bits' mantissa, as the tensor cores take bf16
                    }
                }
            const uint8_t* sv = st + 16 * Geo::ROW;
#pragma unroll
            for (int c = 0; c < VC; c++) {
                unsigned w[4][VB / 4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if constexpr (VB == 16) {
                        const uint4 x = *reinterpret_cast<const uint4*>(sv + (j * VC + c) * 512 + lane * 16);
                        w[j][0] = x.x, w[j][1] = x.y, w[j][2] = x.z, w[j][3] = x.w;
                    } else {
                        const uint2 x = *reinterpret_cast<const uint2*>(sv + (j * VC + c) * 256 + lane * 8);
                        w[j][0] = x.x, w[j][1] = x.y;
                    }
                }
#pragma unroll
                for (int q = 0; q < VB / 4; q++) {
                    if constexpr (F8) {
                        // bytes of positions (2t, 2t + 1) and (2t + 8, 2t + 9) interleaved: four dimensions
                        const unsigned a = __byte_perm(w[0][q], w[1][q], 0x5140), a2 = __byte_perm(w[0][q], w[1][q], 0x7362);
                        const unsigned d = __byte_perm(w[2][q], w[3][q], 0x5140), d2 = __byte_perm(w[2][q], w[3][q], 0x7362);
                        const int n = c * VB + 4 * q;
                        mma16816<true>(acc[n], pa[0], pa[1], pa[2], pa[3], f16x2_of(a), f16x2_of(d));
                        mma16816<true>(acc[n + 1], pa[0], pa[1], pa[2], pa[3], f16x2_of(a >> 16), f16x2_of(d >> 16));
                        mma16816<true>(acc[n + 2], pa[0], pa[1], pa[2], pa[3], f16x2_of(a2), f16x2_of(d2));
                        mma16816<true>(acc[n + 3], pa[0], pa[1], pa[2], pa[3], f16x2_of(a2 >> 16), f16x2_of(d2 >> 16));
                    } else {
                        const int n = c * (VB / 2) + 2 * q;
                        mma16816<false>(acc[n], pa[0], pa[1], pa[2], pa[3], __byte_perm(w[0][q], w[1][q], 0x5410),
                                        __byte_perm(w[2][q], w[3][q], 0x5410));
                        mma16816<false>(acc[n + 1], pa[0], pa[1], pa[2], pa[3], __byte_perm(w[0][q], w[1][q], 0x7632),
                                        __byte_perm(w[2][q], w[3][q], 0x7632));
                    }
                }
            }
            if constexpr (F8) __syncwarp();  // exponents read before a later group overwrites them
        }
        cp_wait<0>();

        // ---- the CTA's partial: its warps' joined in warp order ----
#pragma unroll
        for (int half = 0; half < 2; half++) {
            l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
            l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
            if (t == 0) {
                mls[warp][g + 8 * half][0] = m[half];
                mls[warp][g + 8 * half][1] = l[half];
            }
        }
        __syncthreads();  // every warp is done with the ring
        float* merge = reinterpret_cast<float*>(smem);  // [warp][16][PAD]
        {
            const float un = F8 ? (X < -500 ? 0.0f : exp_byte(static_cast<unsigned>(X))) : 1.0f;
            // column n of the tile c (VB bytes a lane: NV dimensions) is dimension c * 8 NV + n NV + i
            constexpr int NV = F8 ? VB : VB / 2;
#pragma unroll
            for (int half = 0; half < 2; half++) {
                if (g + 8 * half >= rows) continue;
                float* row = merge + (warp * kDecRows + g + 8 * half) * PAD;
#pragma unroll
                for (int c = 0; c < VC; c++)
#pragma unroll
                    for (int col = 0; col < 2; col++)
#pragma unroll
                        for (int i = 0; i < NV; i += 4)
                            *reinterpret_cast<float4*>(row + c * 8 * NV + (2 * t + col) * NV + i) =
                                make_float4(acc[c * NV + i][2 * half + col] * un, acc[c * NV + i + 1][2 * half + col] * un,
                                            acc[c * NV + i + 2][2 * half + col] * un, acc[c * NV + i + 3][2 * half + col] * un);
            }
        }
        __syncthreads();
        const int first = dec_owner(W, pair_first, S), final_cta = dec_owner(W, pair_end - 1, S);
        const int parts = final_cta - first + 1;
        const int quads = rows * (D / 4);
        float* my_part = ws.part + static_cast<int64_t>(2 * cta + (lo == pair_first ? 1 : 0)) * ws.rows * PAD;
        bool odd = false;
        auto finish = [&](int r, int d, float4 o, float lsum) {
            const int token = r / p.G;
            const bool sees = sq.len - sq.n + token >= 0 && sq.len > 0;
            const float inv = sees ? 1.0f / lsum : 0.0f;
            o.x *= inv, o.y *= inv, o.z *= inv, o.w *= inv;
            if (!sees) o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            odd |= !(fabsf(o.x) + fabsf(o.y) + fabsf(o.z) + fabsf(o.w) <= 3.4e38f);
            uint2 v;
            v.x = pack_bf16(o.x, o.y);
            v.y = pack_bf16(o.z, o.w);
            *reinterpret_cast<uint2*>(p.out + static_cast<int64_t>(sq.q0 + token) * p.out_stride +
                                      static_cast<int64_t>(kvh * p.G + r - token * p.G) * D + d) = v;
        };
        for (int o = tid; o < quads; o += kDecThreads) {
            const int r = o / (D / 4), d = (o % (D / 4)) * 4;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < kDecWarps; w++) M = fmaxf(M, mls[w][r][0]);
            const float base = M == -INFINITY ? 0.0f : M;
            float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            float ls = 0.0f;
#pragma unroll
            for (int w = 0; w < kDecWarps; w++) {
                const float f = exp2_fast(mls[w][r][0] - base);
                const float4 v = *reinterpret_cast<const float4*>(merge + (w * kDecRows + r) * PAD + d);
                a.x = fmaf(f, v.x, a.x), a.y = fmaf(f, v.y, a.y), a.z = fmaf(f, v.z, a.z), a.w = fmaf(f, v.w, a.w);
                ls = fmaf(f, mls[w][r][1], ls);
            }
            if (parts == 1) {
                finish(r, d, a, ls);
            } else {
                *reinterpret_cast<float4*>(my_part + r * PAD + d) = a;
                if (d == 0) *reinterpret_cast<float2*>(my_part + r * PAD + D) = make_float2(M, ls);
            }
        }
        if (parts > 1) {
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                unsigned* counter = ws.counters + first;  // a CTA starts at most one (sequence, kv head) that it does not end
                last = atomicAdd(counter, 1u) == static_cast<unsigned>(parts - 1);
                if (last) *counter = 0u;
            }
            __syncthreads();
            if (last) {
                __threadfence();
                auto part_of = [&](int i) {
                    // the first CTA's blocks of the pair are its last segment unless the pair starts it
                    return ws.part + static_cast<int64_t>(2 * (first + i) + (i == 0 ? 1 : 0)) * ws.rows * PAD;
                };
                for (int o = tid; o < quads; o += kDecThreads) {
                    const int r = o / (D / 4), d = (o % (D / 4)) * 4;
                    float M = -INFINITY;
#pragma unroll 4
                    for (int i = 0; i < parts; i++) M = fmaxf(M, __ldcg(part_of(i) + r * PAD + D));
                    const float base = M == -INFINITY ? 0.0f : M;
                    float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    float ls = 0.0f;
#pragma unroll 4
                    for (int i = 0; i < parts; i++) {
                        const float* pr = part_of(i) + r * PAD;
                        const float2 ml = __ldcg(reinterpret_cast<const float2*>(pr + D));
                        const float f = exp2_fast(ml.x - base);
                        const float4 v = __ldcg(reinterpret_cast<const float4*>(pr + d));
                        a.x = fmaf(f, v.x, a.x), a.y = fmaf(f, v.y, a.y), a.z = fmaf(f, v.z, a.z), a.w = fmaf(f, v.w, a.w);
                        ls = fmaf(f, ml.y, ls);
                    }
                    finish(r, d, a, ls);
                }
            }
        }
        // A value that is not finite, behind some row's mask, reaches that row as 0 * inf through the
        // matrix product: then every row is done again in plain loops over what it sees.
        if (__syncthreads_or(odd) && sq.n > 1) {
            for (int r = warp; r < rows; r += kDecWarps) {
                const int token = r / p.G, head = kvh * p.G + r - token * p.G;
                const int see = max(0, min(sq.len, sq.len - sq.n + token + 1));
                float mm, ll, a[D / 32];
                attend_row<KIND, D>(p, b, sq.q0, sq.q0 + token, head, 0, see, lane, mm, ll, a);
                uint16_t* o = p.out + static_cast<int64_t>(sq.q0 + token) * p.out_stride + static_cast<int64_t>(head) * D + lane * (D / 32);
                const float inv = see > 0 ? 1.0f / ll : 0.0f;
#pragma unroll
                for (int i = 0; i < D / 32; i += 2) *reinterpret_cast<unsigned*>(o + i) = pack_bf16(a[i] * inv, a[i + 1] * inv);
            }
        }
        lo = seg_end;
    }
}

}  // namespace oomb
