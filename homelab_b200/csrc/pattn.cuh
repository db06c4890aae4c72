// pattn.cuh - causal grouped-query attention of a step's new tokens over a paged cache,
// or over the step's own packed rows (whole prompts).
//
// New token i of sequence b (n_b of them, kv_len = len) sees the first
// vis = len - n_b + i + 1 positions, clamped to [0, len]:
//   out[i, h, :] = sum_j<vis e^(scale q.k_j - m) v_j / sum_j<vis e^(scale q.k_j - m),
// m the largest score of the row; a row that sees nothing gets zeros.  Scores, maxima,
// sums and outputs are kept in fp32; the output is rounded once to bf16.
#pragma once

#include "paged.cuh"

namespace oomb {

struct PattnParams {
    const uint16_t* q;      // bf16 [T][H][D]
    int64_t q_stride;       // elements from token to token
    uint16_t* out;          // bf16 [T][H][D]
    int64_t out_stride;
    const int32_t* q_start;  // [B + 1], or null: one token a sequence
    const int32_t* kv_len;   // [B]; null (packed rows): the sequence's own tokens
    int B, T, H, Hkv, G, max_q;
    int kv_max;
    float scale_log2;        // scale * log2(e)
    KvView kv;
    unsigned* err;
};

enum : int { KV_ROWS = 0, KV_BF16 = 1, KV_E4M3 = 2 };

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 2^e, e in [-126, 127].
__device__ __forceinline__ float power_of(int e) { return __int_as_float((e + 127) << 23); }

// Lane's D / 32 values of key (or value) row j of sequence b, kv head h, as fp32; a bad
// block table entry reads as zeros.
template <int KIND, int D>
__device__ __forceinline__ void kv_row(const PattnParams& p, bool value, int b, int base_row, int h, int j, int lane, float (&f)[D / 32]) {
    constexpr int E = D / 32;
    const uint8_t* base = value ? p.kv.v : p.kv.k;
    int64_t o;
    float s = 1.0f;
    if constexpr (KIND == KV_ROWS) {
        o = static_cast<int64_t>(base_row + j) * (value ? p.kv.v_stride : p.kv.k_stride) + static_cast<int64_t>(h) * D;
    } else {
        const int page = __ldcg(p.kv.table + static_cast<int64_t>(b) * p.kv.table_stride + (j >> p.kv.page_log2));
        const int slot = j & ((1 << p.kv.page_log2) - 1);
        if (page < 0 || page >= p.kv.num_pages) {
            if (lane == 0) record_error(p.err, ERR_KV_TABLE);
#pragma unroll
            for (int i = 0; i < E; i++) f[i] = 0.0f;
            return;
        }
        o = page * p.kv.page_stride + ((static_cast<int64_t>(h) << p.kv.page_log2) + slot) * D;
        if constexpr (KIND == KV_E4M3)
            s = exp_byte((value ? p.kv.ve : p.kv.ke)[page * p.kv.exp_stride + (static_cast<int64_t>(h) << p.kv.page_log2) + slot]);
    }
    o += lane * E;
#pragma unroll
    for (int i = 0; i < E; i += 2) {
        if constexpr (KIND == KV_E4M3) {
            const float2 d = e4m3x2_to_float2(*reinterpret_cast<const unsigned short*>(base + o + i));
            f[i] = d.x * s;
            f[i + 1] = d.y * s;
        } else {
            const unsigned w = *reinterpret_cast<const unsigned*>(base + 2 * (o + i));
            f[i] = __uint_as_float(w << 16);
            f[i + 1] = __uint_as_float(w & 0xffff0000u);
        }
    }
}

// Whether a value row of the positions [j0, j1) holds something that is not finite (for the whole warp).
template <int KIND, int D>
__device__ __noinline__ bool odd_values(const PattnParams& p, int b, int base_row, int h, int j0, int j1, int lane) {
    bool odd = false;
    for (int j = j0; j < j1; j++) {
        float f[D / 32];
        kv_row<KIND, D>(p, true, b, base_row, h, j, lane, f);
#pragma unroll
        for (int i = 0; i < D / 32; i++) odd |= !(fabsf(f[i]) <= 3.4e38f);
    }
    return __any_sync(0xffffffffu, odd);
}

// One query row over positions [j0, j1) (of packed rows from base_row on, or of sequence b's pages) by one warp, in plain fp32 loops: the running
// maximum m (in units of log2), sum l and unnormalised output acc of the row.  `beat` moves on the way, for those who wait.
template <int KIND, int D>
__device__ __noinline__ void attend_row(const PattnParams& p, int b, int base_row, int token, int head, int j0, int j1, int lane, unsigned* beat, float& m,
                                        float& l, float (&acc)[D / 32]) {
    constexpr int E = D / 32;
    float q[E];
    const uint16_t* qp = p.q + static_cast<int64_t>(token) * p.q_stride + static_cast<int64_t>(head) * D + lane * E;
#pragma unroll
    for (int i = 0; i < E; i++) {
        q[i] = bf16_bits_to_float(qp[i]) * p.scale_log2;
        acc[i] = 0.0f;
    }
    m = -INFINITY;
    l = 0.0f;
    for (int j = j0; j < j1; j++) {
        if ((j & 1023) == 0 || j == j0) {
            if (lane == 0) atomicAdd(beat, 1u);
        }
        float k[E], v[E];
        kv_row<KIND, D>(p, false, b, base_row, head / p.G, j, lane, k);
        kv_row<KIND, D>(p, true, b, base_row, head / p.G, j, lane, v);
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < E; i++) s = fmaf(q[i], k[i], s);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        const float mn = fmaxf(m, s);
        const float base = mn == -INFINITY ? 0.0f : mn;
        const float c = exp2_fast(m - base), e = exp2_fast(s - base);
        l = fmaf(l, c, e);
#pragma unroll
        for (int i = 0; i < E; i++) acc[i] = fmaf(acc[i], c, e * v[i]);
        m = mn;
    }
}

}  // namespace oomb
