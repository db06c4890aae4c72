// paged.cuh - rotary positions, and a paged key/value cache in bf16 or in 8 bits: its
// write, fused with the rotation, and its read-back.
//
// A pool holds num_pages pages; a page holds page_size positions of every kv head, row
// (page, head, slot) of head_dim values contiguous, so the positions of one (page, head)
// are one run of page_size * head_dim values that attention streams.  Row b of the block
// table names the pages of sequence b in order: position j sits in page table[b][j / ps]
// at slot j % ps.  Three equal ways to say where a step's tokens go serve every kernel
// here: token t of the packed step belongs to the sequence b with
// q_start[b] <= t < q_start[b + 1], and its position is kv_len[b] - n_b + (t - q_start[b]),
// n_b = q_start[b + 1] - q_start[b] (kv_len counts the new tokens).
//
// 8-bit rows: x = e4m3 * 2^e with one e per (position, head), kept as the byte e + 127.
// A power of two keeps every code's product exact in bf16 and in fp32, so no reader
// rounds again.  e is the least with amax * r <= 448 * 2^e over the finite values of the
// row BEFORE rotation, r = sqrt(2) * mscale for a rotated row (a rotation grows a value
// by at most sqrt(2)) and 1 otherwise: comparing the input's largest value with a
// constant is exact, so the byte does not depend on how the angles were rounded.
// e4m3 being a floating type, the factor sqrt(2) costs no precision above 2^-6 * 2^e.
// Infinities and NaN become the NaN code; e is clamped to [-100, 120], and codes to what an fp32 number can stand for.
//
// Angles: the frequency of a pair is kept as turns per position in units of 2^-64; a
// position times it modulo 2^64 is the exact phase, of which 32 bits go to sincospif:
// no loss at far positions and no table to read (an fp32 product loses 1e-2 rad at
// position 100,000).
//
// Bound: HBM for prompts (each value read once and written once), launch latency for
// decode steps.  One CTA takes `tpb` tokens: their angles go through shared memory once
// and serve all heads; a row is rotated by head_dim / 16 threads with two 8-value
// chunks each, a pair's two halves in the same thread, so a rotation may be in place.
#pragma once

#include "common.cuh"

namespace oomb {

enum : unsigned {
    ERR_KV_TABLE = 0x900,  // a block table entry was outside the pool (its positions skipped, or read as zeros)
    ERR_KV_SEQ = 0x910,    // q_start or kv_len out of range (the sequence clamped or skipped)
};

// Where attention finds keys and values: packed rows of the step, or pages.
struct KvView {
    const uint8_t* k;
    const uint8_t* v;
    const uint8_t* ke;      // exponent bytes [pages][kv_heads][page], e4m3 pools only
    const uint8_t* ve;
    int64_t page_stride;    // elements from page to page (exponents: exp_stride)
    int64_t exp_stride;
    const int32_t* table;
    int table_stride;       // entries from one sequence's row to the next
    int max_pages;          // entries of a row in use at most
    int num_pages;
    int page_log2;
    int Hkv;
    int64_t k_stride, v_stride;  // packed rows: elements from token to token
    int seq_rows;                // packed rows: sequence b's keys begin at row b * seq_rows; 0: at its first token
};

// The sequence that token t belongs to: the number of b with q_start[b + 1] <= t, by a
// 32-way search of one warp (B <= 32: one load).  Every lane gets it; B when t is behind
// the last sequence.
__device__ __forceinline__ int find_sequence(const int32_t* q_start, int B, int t, int lane) {
    int lo = 0, n = B;
    while (n > 0) {
        const int step = (n + 31) / 32;
        const int i = lo + (lane + 1) * step - 1;
        const bool past = i < lo + n && __ldcg(q_start + i + 1) <= t;
        const int c = __popc(__ballot_sync(0xffffffffu, past));
        const int end = lo + n;
        lo += c * step;
        n = min(step, end - lo);
        if (step == 1) break;
    }
    return lo;
}

struct Seq {
    int q0, n, len;  // first packed token, new tokens, cached positions with them
};

// Sequence b's numbers, forced into range (and the device error word set) where they are
// not: 0 <= q0 <= q0 + n <= T, 0 <= len <= kv_max.
__device__ __forceinline__ Seq read_seq(const int32_t* q_start, const int32_t* kv_len, int b, int T, int kv_max,
                                        unsigned* err) {
    Seq s;
    const int a = q_start ? __ldcg(q_start + b) : b, e = q_start ? __ldcg(q_start + b + 1) : b + 1;
    s.q0 = max(0, min(a, T));
    s.n = max(0, min(e, T) - s.q0);
    const int len = kv_len ? __ldcg(kv_len + b) : s.n;
    s.len = max(0, min(len, kv_max));
    if (a < 0 || e < a || e > T || len < s.n || len > kv_max) record_error(err, ERR_KV_SEQ);
    return s;
}

// ---- rotation and append -------------------------------------------------------------

constexpr int kRowsThreads = 256;
// Tokens of a CTA.  8,192 new tokens of 32 query heads over 8, D = 128 (101 MB read, 101 written), take 46.0 us with one,
// 38.8 with two and 40.0 with three or four; rotation alone of 9,391 fp32 tokens of 32 heads (308 MB) 47.7, 49.2, 50.4 and 51.8.
constexpr int kRowsMaxTpb = 2;
constexpr int kRopeMaxPairs = 64;  // head_dim / 2

struct RowsParams {
    const void *q, *k, *v;  // q null: none; k null: rotation alone
    int64_t qs, ks, vs;     // elements from token to token
    void* qo;
    int64_t qos;
    int qo_bf16;
    int Hq, Hkv;
    const uint64_t* turns;  // null: no rotation
    int rot, interleaved;
    float mscale;
    float k_limit;          // e4m3: 448, or 448 / (sqrt(2) * mscale) of rotated keys
    const int32_t* positions;  // rotation alone: [T]
    const int32_t* q_start;    // append: [B + 1], or null for one token a sequence
    const int32_t* kv_len;
    int B, T, tpb;
    KvView kv;
    uint8_t *ko, *vo, *keo, *veo;  // the pool, to be written
    unsigned* err;
};

template <bool BF16>
__device__ __forceinline__ void load8(const void* base, int64_t idx, float (&f)[8]) {
    if constexpr (BF16) {
        const uint4 w = __ldcg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + idx));
        const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f[2 * i] = __uint_as_float(u[i] << 16);
            f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    } else {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + idx);
        const float4 a = __ldcg(p), b = __ldcg(p + 1);
        f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    }
}

__device__ __forceinline__ void store8(void* base, int64_t idx, bool bf16, const float (&f)[8]) {
    if (bf16) {
        uint4 o;
        unsigned* w = reinterpret_cast<unsigned*>(&o);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
            w[i] = *reinterpret_cast<const unsigned*>(&h);
        }
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + idx) = o;
    } else {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + idx);
        p[0] = make_float4(f[0], f[1], f[2], f[3]);
        p[1] = make_float4(f[4], f[5], f[6], f[7]);
    }
}

// The least e with amax <= limit * 2^e (amax, limit finite; 0 for a zero row), clamped.
__device__ __forceinline__ int row_exponent(float amax, float limit) {
    const unsigned a = __float_as_uint(amax), l = __float_as_uint(limit);
    const int e = static_cast<int>(a >> 23) - static_cast<int>(l >> 23) + ((a & 0x7fffffu) > (l & 0x7fffffu) ? 1 : 0);
    return amax > 0.0f ? max(-100, min(120, e)) : 0;
}

// Finite values of a row with the largest exponent, 120, held within 240 * 2^120: the codes above stand for 2^128 and more, which no
// fp32 number is (2^128 itself is off by 2^-4 so, a rounding's most).
__device__ __forceinline__ void hold_finite(float (&f)[8]) {
    constexpr float kTop = 3.1901471898837980e38f;  // 15 * 2^124
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (fabsf(f[i]) > kTop && fabsf(f[i]) <= 3.4028235e38f) f[i] = copysignf(kTop, f[i]);
}

// Eight values times 2^-e as e4m3 codes; non-finite values become the NaN code.
__device__ __forceinline__ uint2 codes8(const float (&f)[8], float inv) {
    unsigned w[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        unsigned r = 0;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            float a = f[4 * i + 2 * j] * inv, b = f[4 * i + 2 * j + 1] * inv;
            a = fabsf(a) <= 3.4e38f ? a : __uint_as_float(0x7fffffffu);
            b = fabsf(b) <= 3.4e38f ? b : __uint_as_float(0x7fffffffu);
            unsigned short c;
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(c) : "f"(b), "f"(a));
            r |= static_cast<unsigned>(c) << (16 * j);
        }
        w[i] = r;
    }
    return make_uint2(w[0], w[1]);
}

// CACHE: -1 rotation alone, 0 bf16 pool, 1 e4m3 pool.  Six CTAs to an SM (40 registers): the append above takes 45 us with
// five of 48 registers and 41 with seven of 36.
template <bool XBF16, int D, int CACHE>
__global__ void __launch_bounds__(kRowsThreads, 6) rows_kernel(const RowsParams p) {
    constexpr int TEAM = D / 16;  // threads of a row
    constexpr int SLOTS = kRowsThreads / TEAM;
    __shared__ __align__(16) float cs[kRowsMaxTpb][2][kRopeMaxPairs];
    __shared__ int tok_ok[kRowsMaxTpb], tok_pos[kRowsMaxTpb];
    __shared__ int64_t tok_row[kRowsMaxTpb], tok_exp[kRowsMaxTpb];
    const int t0 = blockIdx.x * p.tpb, nt = min(p.tpb, p.T - t0);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    pdl_launch_dependents();
    if (warp < nt) {
        const int t = t0 + warp;
        int pos = 0;
        bool ok = true;
        int64_t row = -1, ex = -1;
        if constexpr (CACHE < 0) {
            pos = __ldcg(p.positions + t);
        } else {
            const int b = p.q_start ? find_sequence(p.q_start, p.B, t, lane) : t;
            ok = b < p.B && (!p.q_start || t >= __ldcg(p.q_start));
            if (ok) {
                const int kv_max = p.kv.max_pages << p.kv.page_log2;
                const int q0 = p.q_start ? __ldcg(p.q_start + b) : b, q1 = p.q_start ? __ldcg(p.q_start + b + 1) : b + 1;
                pos = __ldcg(p.kv_len + b) - (q1 - q0) + (t - q0);
                if (pos < 0 || pos >= kv_max) {
                    ok = false;  // nowhere to write: the token is skipped
                    if (lane == 0) record_error(p.err, ERR_KV_SEQ);
                } else {
                    const int page = __ldcg(p.kv.table + static_cast<int64_t>(b) * p.kv.table_stride + (pos >> p.kv.page_log2));
                    const int slot = pos & ((1 << p.kv.page_log2) - 1);
                    if (page < 0 || page >= p.kv.num_pages) {
                        if (lane == 0) record_error(p.err, ERR_KV_TABLE);
                    } else {
                        row = page * p.kv.page_stride + static_cast<int64_t>(slot) * D;
                        ex = page * p.kv.exp_stride + slot;
                    }
                }
            }
        }
        if (lane == 0) {
            tok_ok[warp] = ok;
            tok_pos[warp] = pos;
            tok_row[warp] = row;
            tok_exp[warp] = ex;
        }
    }
    if (p.turns) {
        __syncthreads();
        const int pairs = p.rot / 2;
        for (int i = threadIdx.x; i < nt * pairs; i += kRowsThreads) {
            const int a = i / pairs, f = i - a * pairs;
            const uint64_t phase = static_cast<uint64_t>(static_cast<int64_t>(tok_pos[a])) * __ldg(p.turns + f) + 0x80000000ull;
            float s, c;
            sincospif(static_cast<float>(static_cast<int>(phase >> 32)) * 4.656612873077393e-10f, &s, &c);  // 2^-31
            cs[a][0][f] = c * p.mscale;
            cs[a][1][f] = s * p.mscale;
        }
    }
    __syncthreads();

    const int R = p.Hq + 2 * p.Hkv, slot = threadIdx.x / TEAM, t8 = threadIdx.x % TEAM;
    const int total = nt * R;
    int a = slot / R, rr = slot - a * R;  // token of the CTA, row of the token
    for (int r0 = 0; r0 < total; r0 += SLOTS, rr += SLOTS) {
        const bool in = r0 + slot < total;
        while (rr >= R) {
            rr -= R;
            a = min(a + 1, kRowsMaxTpb - 1);  // past the last token nothing is done, but its flag is read
        }
        const bool is_q = rr < p.Hq, is_k = !is_q && rr < p.Hq + p.Hkv;
        const int h = is_q ? rr : is_k ? rr - p.Hq : rr - p.Hq - p.Hkv;
        const bool ok = in && tok_ok[a];
        const bool turn = p.turns && (is_q || is_k);
        // this thread's two chunks of eight values: the two halves of its pairs when the halves
        // of a rotated row pair up, else any two
        int ca = t8, cb = t8 + TEAM;
        const int nr = p.rot / 16;
        if (turn && !p.interleaved) {
            if (t8 < nr) {
                cb = t8 + nr;
            } else {
                ca = 2 * nr + (t8 - nr);
                cb = ca + (TEAM - nr);
            }
        }
        float x[8] = {}, y[8] = {};
        if (ok) {
            const void* src = is_q ? p.q : is_k ? p.k : p.v;
            const int64_t base = static_cast<int64_t>(t0 + a) * (is_q ? p.qs : is_k ? p.ks : p.vs) + static_cast<int64_t>(h) * D;
            load8<XBF16>(src, base + ca * 8, x);
            load8<XBF16>(src, base + cb * 8, y);
        }
        float amax = 0.0f;
        if constexpr (CACHE == 1) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float u = fabsf(x[i]), w = fabsf(y[i]);
                amax = fmaxf(amax, fmaxf(u <= 3.4028235e38f ? u : 0.0f, w <= 3.4028235e38f ? w : 0.0f));
            }
#pragma unroll
            for (int o = 1; o < TEAM; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        }
        if (!ok) continue;
        if (turn) {
            const float* c = cs[a][0];
            const float* s = cs[a][1];
            if (p.interleaved) {
                const float4 ca4 = *reinterpret_cast<const float4*>(c + ca * 4), sa4 = *reinterpret_cast<const float4*>(s + ca * 4);
                const float4 cb4 = *reinterpret_cast<const float4*>(c + cb * 4), sb4 = *reinterpret_cast<const float4*>(s + cb * 4);
                const float c1[4] = {ca4.x, ca4.y, ca4.z, ca4.w}, s1[4] = {sa4.x, sa4.y, sa4.z, sa4.w};
                const float c2[4] = {cb4.x, cb4.y, cb4.z, cb4.w}, s2[4] = {sb4.x, sb4.y, sb4.z, sb4.w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (ca * 8 < p.rot) {  // rot is a multiple of 16: a chunk turns as a whole
                        const float u = x[2 * i], w = x[2 * i + 1];
                        x[2 * i] = u * c1[i] - w * s1[i];
                        x[2 * i + 1] = w * c1[i] + u * s1[i];
                    }
                    if (cb * 8 < p.rot) {
                        const float u = y[2 * i], w = y[2 * i + 1];
                        y[2 * i] = u * c2[i] - w * s2[i];
                        y[2 * i + 1] = w * c2[i] + u * s2[i];
                    }
                }
            } else if (t8 < nr) {
#pragma unroll
                for (int i = 0; i < 8; i += 4) {
                    const float4 c4 = *reinterpret_cast<const float4*>(c + t8 * 8 + i), s4 = *reinterpret_cast<const float4*>(s + t8 * 8 + i);
                    const float cc[4] = {c4.x, c4.y, c4.z, c4.w}, ss[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const float u = x[i + k], w = y[i + k];
                        x[i + k] = u * cc[k] - w * ss[k];
                        y[i + k] = w * cc[k] + u * ss[k];
                    }
                }
            }
        }
        if (is_q) {
            const int64_t o = static_cast<int64_t>(t0 + a) * p.qos + static_cast<int64_t>(h) * D;
            store8(p.qo, o + ca * 8, p.qo_bf16, x);
            store8(p.qo, o + cb * 8, p.qo_bf16, y);
        } else if constexpr (CACHE >= 0) {
            if (tok_row[a] < 0) continue;
            const int64_t o = tok_row[a] + (static_cast<int64_t>(h) * D << p.kv.page_log2);
            uint8_t* pool = is_k ? p.ko : p.vo;
            if constexpr (CACHE == 0) {
                store8(pool, o + ca * 8, true, x);
                store8(pool, o + cb * 8, true, y);
            } else {
                const int e = row_exponent(amax, is_k ? p.k_limit : 448.0f);
                const float inv = __int_as_float((127 - e) << 23);
                if (e == 120) {
                    hold_finite(x);
                    hold_finite(y);
                }
                *reinterpret_cast<uint2*>(pool + o + ca * 8) = codes8(x, inv);
                *reinterpret_cast<uint2*>(pool + o + cb * 8) = codes8(y, inv);
                if (t8 == 0)
                    (is_k ? p.keo : p.veo)[tok_exp[a] + (static_cast<int64_t>(h) << p.kv.page_log2)] = static_cast<uint8_t>(e + 127);
            }
        }
    }
}

// ---- read-back -----------------------------------------------------------------------

constexpr int kReadThreads = 256;
// Tokens of a CTA, one warp each for the lookup, and a thread's chunks under way: 2,047 e4m3 positions of 8 heads, D = 128, and
// 42,385 bf16 ones take 6.0 and 62.4 us with four and two, 6.9 and 62.9 with eight and four, 6.9 and 65.4 with eight and two,
// 7.5 and 65.6 with four and four, 5.8 and 66.0 with two and two.
constexpr int kReadTokens = 4, kReadAhead = 2;

struct ReadParams {
    KvView kv;
    const int32_t* q_start;
    const int32_t* kv_len;
    int B, T;
    void *ko, *vo;
    int out_bf16;
    int64_t out_stride;
    unsigned* err;
};

// 2^(byte - 127); 0 for byte 0.
__device__ __forceinline__ float exp_byte(unsigned e) { return __uint_as_float(e << 23); }

// Rows of the packed positions, keys and values: out[t][h][:] = the row's values.  A
// thread moves 8 values: 16-byte stores of consecutive lanes are contiguous.
template <bool FP8, int D>
__global__ void __launch_bounds__(kReadThreads) read_kernel(const ReadParams p) {
    __shared__ int64_t tok_row[kReadTokens], tok_exp[kReadTokens];
    const int t0 = blockIdx.x * kReadTokens, nt = min(kReadTokens, p.T - t0);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    pdl_launch_dependents();
    if (warp < nt) {
        const int t = t0 + warp;
        const int b = p.q_start ? find_sequence(p.q_start, p.B, t, lane) : t;
        int64_t row = -2, ex = 0;  // -2: leave the output row as it was; -1: zeros
        if (b < p.B && (!p.q_start || t >= __ldcg(p.q_start))) {
            const int kv_max = p.kv.max_pages << p.kv.page_log2;
            const int q0 = p.q_start ? __ldcg(p.q_start + b) : b, q1 = p.q_start ? __ldcg(p.q_start + b + 1) : b + 1;
            const int pos = __ldcg(p.kv_len + b) - (q1 - q0) + (t - q0);
            row = -1;
            if (pos < 0 || pos >= kv_max) {
                if (lane == 0) record_error(p.err, ERR_KV_SEQ);
            } else {
                const int page = __ldcg(p.kv.table + static_cast<int64_t>(b) * p.kv.table_stride + (pos >> p.kv.page_log2));
                const int slot = pos & ((1 << p.kv.page_log2) - 1);
                if (page < 0 || page >= p.kv.num_pages) {
                    if (lane == 0) record_error(p.err, ERR_KV_TABLE);
                } else {
                    row = page * p.kv.page_stride + static_cast<int64_t>(slot) * D;
                    ex = page * p.kv.exp_stride + slot;
                }
            }
        }
        if (lane == 0) {
            tok_row[warp] = row;
            tok_exp[warp] = ex;
        }
    }
    __syncthreads();
    // Chunks of 8 values, kReadAhead under way at once: (token, keys or values, head, chunk).
    const int per_row = p.kv.Hkv * (D / 8), per_tok = 2 * per_row, total = nt * per_tok;
    constexpr int N = kReadAhead;
    for (int i0 = threadIdx.x; i0 < total; i0 += N * kReadThreads) {
        uint4 w[N];
        unsigned e[N];
        int64_t to[N];
        bool is_v[N], leave[N];
#pragma unroll
        for (int k = 0; k < N; k++) {
            const int i = i0 + k * kReadThreads;
            w[k] = make_uint4(0u, 0u, 0u, 0u);
            e[k] = 127u;
            leave[k] = true;
            if (i >= total) continue;
            const int a = i / per_tok, rest = i - a * per_tok;
            is_v[k] = rest >= per_row;
            const int c = is_v[k] ? rest - per_row : rest, h = c / (D / 8), c8 = (c % (D / 8)) * 8;
            const int64_t row = tok_row[a];
            if (row == -2) continue;
            leave[k] = false;
            to[k] = static_cast<int64_t>(t0 + a) * p.out_stride + h * D + c8;
            if (row < 0) continue;
            const int64_t o = row + (static_cast<int64_t>(h) * D << p.kv.page_log2) + c8;
            const uint8_t* pool = is_v[k] ? p.kv.v : p.kv.k;
            if constexpr (FP8) {
                const uint2 u = __ldcs(reinterpret_cast<const uint2*>(pool + o));
                w[k].x = u.x;
                w[k].y = u.y;
                e[k] = (is_v[k] ? p.kv.ve : p.kv.ke)[tok_exp[a] + (static_cast<int64_t>(h) << p.kv.page_log2)];
            } else {
                w[k] = __ldcs(reinterpret_cast<const uint4*>(pool + 2 * o));
            }
        }
#pragma unroll
        for (int k = 0; k < N; k++) {
            if (leave[k]) continue;
            float f[8];
            if constexpr (FP8) {
                const float s = exp_byte(e[k]);
                const unsigned u[2] = {w[k].x, w[k].y};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float2 d = e4m3x2_to_float2(static_cast<unsigned short>(u[j / 2] >> (16 * (j & 1))));
                    f[2 * j] = d.x * s;
                    f[2 * j + 1] = d.y * s;
                }
            } else {
                if (p.out_bf16) {
                    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(is_v[k] ? p.vo : p.ko) + to[k]) = w[k];
                    continue;
                }
                const unsigned u[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    f[2 * j] = __uint_as_float(u[j] << 16);
                    f[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
                }
            }
            store8(is_v[k] ? p.vo : p.ko, to[k], p.out_bf16, f);
        }
    }
}

// ---- conversion of a call's codes ------------------------------------------------------

constexpr int kExpandTokens = 8;  // positions of a CTA

struct ExpandParams {
    KvView kv;
    const int32_t* q_start;
    const int32_t* kv_len;
    int B, T, kv_max;
    uint16_t *ko, *vo;  // [B * kv_max][kv_heads][D]
    unsigned* err;
};

// The cached rows of every sequence as bf16 (a code times a power of two is exact there), position j of sequence b at row
// b * kv_max + j: for attention whose query tiles would each convert them again.  A position's page is looked up once a
// CTA; eight values a thread, four loads under way.
template <int D>
__global__ void __launch_bounds__(kReadThreads) expand_kernel(const ExpandParams p) {
    __shared__ int64_t row[kExpandTokens], ex[kExpandTokens];
    pdl_wait();
    pdl_launch_dependents();
    const int b = blockIdx.y, j0 = blockIdx.x * kExpandTokens;
    const Seq s = read_seq(p.q_start, p.kv_len, b, p.T, p.kv_max, nullptr);
    const int nt = s.n > 0 ? min(kExpandTokens, s.len - j0) : 0;
    if (nt <= 0) return;
    if (static_cast<int>(threadIdx.x) < nt) {
        const int j = j0 + threadIdx.x;
        const int page = __ldcg(p.kv.table + static_cast<int64_t>(b) * p.kv.table_stride + (j >> p.kv.page_log2));
        const int slot = j & ((1 << p.kv.page_log2) - 1);
        const bool good = page >= 0 && page < p.kv.num_pages;
        if (!good) record_error(p.err, ERR_KV_TABLE);
        row[threadIdx.x] = good ? page * p.kv.page_stride + static_cast<int64_t>(slot) * D : -1;
        ex[threadIdx.x] = good ? page * p.kv.exp_stride + slot : 0;
    }
    __syncthreads();
    const int per_row = p.kv.Hkv * (D / 8), per_tok = 2 * per_row, total = nt * per_tok;
    constexpr int N = 4;
    for (int i0 = threadIdx.x; i0 < total; i0 += N * kReadThreads) {
        uint2 w[N];
        unsigned e[N];
#pragma unroll
        for (int k = 0; k < N; k++) {
            const int i = i0 + k * kReadThreads;
            w[k] = make_uint2(0u, 0u);
            e[k] = 127u;
            if (i >= total) continue;
            const int a = i / per_tok, rest = i - a * per_tok, c = rest % per_row, h = c / (D / 8), c8 = (c % (D / 8)) * 8;
            if (row[a] < 0) continue;
            const bool v = rest >= per_row;
            w[k] = __ldcs(reinterpret_cast<const uint2*>((v ? p.kv.v : p.kv.k) + row[a] + (static_cast<int64_t>(h) * D << p.kv.page_log2) + c8));
            e[k] = (v ? p.kv.ve : p.kv.ke)[ex[a] + (static_cast<int64_t>(h) << p.kv.page_log2)];
        }
#pragma unroll
        for (int k = 0; k < N; k++) {
            const int i = i0 + k * kReadThreads;
            if (i >= total) continue;
            const int a = i / per_tok, rest = i - a * per_tok, c = rest % per_row;
            const float sc = exp_byte(e[k]);
            const unsigned u[2] = {w[k].x, w[k].y};
            float f[8];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 d = e4m3x2_to_float2(static_cast<unsigned short>(u[j / 2] >> (16 * (j & 1))));
                f[2 * j] = d.x * sc;
                f[2 * j + 1] = d.y * sc;
            }
            store8(rest >= per_row ? p.vo : p.ko, (static_cast<int64_t>(b) * p.kv_max + j0 + a) * p.kv.Hkv * D + c * 8, true, f);
        }
    }
}

}  // namespace oomb
