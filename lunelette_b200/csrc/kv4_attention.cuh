// Causal attention over the paged 4-bit KV cache.
#pragma once
#include "kv4.cuh"

namespace lun {

struct Kv4AttnParams {
    Kv4Cache cache;
    Kv4Rows rows;
    const void *q;
    void *out;
    size_t q_stride, out_stride;
    int query_heads, group;
    float scale;
    int *status;
};

// One warp per (row, query head), 32 keys a step: a lane scores one key, then
// takes D / 32 dims of the weighted sum.
template <int D, typename T>
static __global__ void __launch_bounds__(32) kv4_attention_kernel(Kv4AttnParams p)
{
    using L = Kv4Layout<D>;
    constexpr int per = D / 32;
    const int row = blockIdx.x, head = blockIdx.y, kvh = head / p.group, lane = threadIdx.x;
    __shared__ float qs[D];
    pdl_wait();
    pdl_launch_dependents();
    const int s = kv4_sequence_of_row(p.rows, row);
    const Kv4Sequence q = kv4_sequence(p.rows, s);
    if (!q.ok) {
        if (lane == 0) kv4_report(p.status, kKv4BadRows);
        return;
    }
    if (row < q.first || row >= q.first + q.count) return;
    const int position = q.length - q.count + (row - q.first);
    const T *src = static_cast<const T *>(p.q) + (size_t)row * p.q_stride + (size_t)head * D;
    for (int d = lane; d < D; d += 32) qs[d] = to_float(src[d]) * p.scale;
    __syncwarp();
    float m = -INFINITY, l = 0.0f, o[per] = {};
    const int *table = p.rows.page_tables + s * p.rows.table_stride;
    for (int p0 = 0; p0 <= position; p0 += 32) {
        const uint8_t *block = kv4_block<D>(p.cache, table[p0 / kPage], kvh);
        if (!block) {
            if (lane == 0) kv4_report(p.status, kKv4BadPage);
            continue;
        }
        const int slot = p0 % kPage + lane;
        float score = -INFINITY;
        if (p0 + lane <= position) {
            score = 0.0f;
            for (int w = 0; w < L::words; w++) {
                const uint32_t word = *reinterpret_cast<const uint32_t *>(block + L::k_word(slot, w));
                const float d = __half2float(*reinterpret_cast<const __half *>(block + L::k_scale(slot, w / 4)));
                float sum = 0.0f;
                for (int e = 0; e < 8; e++) sum = fmaf((float)((int)(word >> (4 * e) & 15u) - 8), qs[8 * w + e], sum);
                score = fmaf(d, sum, score);
            }
        }
        const float mx = fmaxf(m, warp_max(score));
        const float corr = m == -INFINITY ? 0.0f : expf(m - mx);
        const float prob = score == -INFINITY ? 0.0f : expf(score - mx);
        m = mx;
        l = l * corr + warp_sum(prob);
        for (int e = 0; e < per; e++) o[e] *= corr;
        for (int j = 0; j < 32 && p0 + j <= position; j++) {
            const float pj = __shfl_sync(0xffffffffu, prob, j);
            for (int e = 0; e < per; e++) {
                const int d = lane * per + e, sl = p0 % kPage + j;
                const uint32_t word = *reinterpret_cast<const uint32_t *>(block + L::v_word(sl, d / 8));
                const float sc = __half2float(*reinterpret_cast<const __half *>(block + L::v_scale(sl, d / 32)));
                o[e] = fmaf(pj, sc * (float)((int)(word >> (4 * (d % 8)) & 15u) - 8), o[e]);
            }
        }
    }
    T *dst = static_cast<T *>(p.out) + (size_t)row * p.out_stride + (size_t)head * D + lane * per;
    for (int e = 0; e < per; e++) dst[e] = from_float<T>(l == 0.0f ? 0.0f : o[e] / l);
}

}  // namespace lun
