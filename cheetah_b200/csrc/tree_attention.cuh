// Attention of drafted nodes over a paged cache.
//
//   o_i = sum_j softmax_j(q_i . k_j / sqrt(D)) v_j
//
// over the context keys and the nodes whose bit is set in row i's mask. One
// CTA per (row, query head): each thread scores one of kTreeKeys keys, then
// thread d accumulates dimension d of the output; online softmax in f32.
#pragma once

#include "common.cuh"

namespace cheetah {

constexpr int kTreeKeys = 128;

struct TreeAttnParams {
    const uint16_t *q;
    long long q_stride;
    int rows;
    const uint16_t *k_pool, *v_pool;
    const int32_t *page_table;
    int max_pages, num_pages, page_tokens;
    const int32_t *seq_lens, *row_starts;
    int batch;
    const unsigned long long *tree_mask;
    int mask_words;
    const int32_t *positions;
    int window;
    int q_heads, kv_heads;
    float scale;
    uint16_t *out;
};

template <int HD>
__global__ void __launch_bounds__(kTreeKeys) tree_attention_rows_kernel(const TreeAttnParams p) {
    __shared__ float prob[kTreeKeys];
    __shared__ long long cell[kTreeKeys];
    __shared__ float red[kTreeKeys / kWarp];
    __shared__ float q_s[HD];
    const int row = blockIdx.x, head = blockIdx.y, tid = threadIdx.x;
    pdl_wait();
    pdl_launch_dependents();
    // Sequence of this row.
    int lo = 0, hi = p.batch;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (p.row_starts[mid + 1] > row) hi = mid;
        else lo = mid + 1;
    }
    if (lo >= p.batch) return;
    const int b = lo, r0 = p.row_starts[b], n = p.row_starts[b + 1] - r0;
    const int len = p.seq_lens[b], ctx = len - n;
    const int kvh = head / (p.q_heads / p.kv_heads);
    const int pos_min = p.window > 0 ? p.positions[row] - p.window : -1;
    if (tid < HD) q_s[tid] = bf16_to_f32(p.q[row * p.q_stride + head * HD + tid]) * p.scale;
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (int k0 = 0; k0 < len && ctx >= 0; k0 += kTreeKeys) {
        const int j = k0 + tid;
        bool seen = j < len;
        if (seen && j >= ctx) {
            const int node = j - ctx;
            seen = node < 64 * p.mask_words && ((p.tree_mask[(long long)row * p.mask_words + node / 64] >> (node % 64)) & 1);
        }
        if (seen && p.window > 0) seen = (j < ctx ? j : p.positions[r0 + j - ctx]) > pos_min;
        long long at = -1;
        if (seen) {
            const int col = j / p.page_tokens;
            const int page = col < p.max_pages ? p.page_table[(long long)b * p.max_pages + col] : -1;
            if (page >= 0 && page < p.num_pages)
                at = (((long long)page * p.kv_heads + kvh) * p.page_tokens + j % p.page_tokens) * HD;
        }
        float s = -INFINITY;
        if (at >= 0) {
            s = 0.0f;
            for (int d = 0; d < HD; ++d) s = fmaf(q_s[d], bf16_to_f32(p.k_pool[at + d]), s);
        }
        const float wm = warp_max(s);
        if (tid % kWarp == 0) red[tid / kWarp] = wm;
        cell[tid] = at;
        __syncthreads();
        const float m_new = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        const float alpha = m_new == -INFINITY ? 1.0f : expf(m - m_new);
        prob[tid] = at >= 0 ? expf(s - m_new) : 0.0f;
        __syncthreads();
        l *= alpha;
        o *= alpha;
        for (int i = 0; i < kTreeKeys; ++i) {
            if (cell[i] < 0) continue;
            l += prob[i];
            if (tid < HD) o = fmaf(prob[i], bf16_to_f32(p.v_pool[cell[i] + tid]), o);
        }
        m = m_new;
        __syncthreads();
    }
    if (tid < HD) p.out[((long long)row * p.q_heads + head) * HD + tid] = f32_to_bf16_rne(l == 0.0f ? 0.0f : o / l);
}

}  // namespace cheetah
