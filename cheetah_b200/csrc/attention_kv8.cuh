// Causal attention of a batch's new rows over an 8-bit paged cache.
//
//   o_i = sum_j softmax_j(q_i . k_j / sqrt(D)) v_j,   k_j = kc_j ks,  v_j = vc_j vs
//
// with e4m3 codes and one scale per 16 cells and head.
//
// A warp takes every fourth key of one row and head.
#pragma once

#include "common.cuh"
#include "kv8.cuh"

namespace cheetah {

struct Kv8AttnParams {
    const uint16_t *q;
    long long q_stride;
    const uint8_t *k_codes, *v_codes;
    const float *k_scales, *v_scales;
    const int32_t *page_table;
    int max_pages, num_pages, page_tokens;
    const int32_t *seq_lens, *row_starts;
    int batch, rows, window, sinks;
    int q_heads, kv_heads;
    float scale_log2;
    uint16_t *out;
};

constexpr int kKv8SimpleWarps = 4;

template <int HD>
__global__ void __launch_bounds__(kKv8SimpleWarps *kWarp) attention_kv8_simple_kernel(const Kv8AttnParams p) {
    constexpr int V = HD / kWarp;
    __shared__ float part_s[kKv8SimpleWarps][HD + 2];
    const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
    const int row = blockIdx.x / p.q_heads, head = blockIdx.x % p.q_heads;
    pdl_wait();
    pdl_launch_dependents();
    if (row >= p.row_starts[p.batch]) return;
    int b = 0, hi = p.batch - 1;
    while (b < hi) {
        const int mid = (b + hi) / 2;
        if (p.row_starts[mid + 1] > row) hi = mid;
        else b = mid + 1;
    }
    const int n = p.row_starts[b + 1] - p.row_starts[b], len = p.seq_lens[b];
    const int pos = len - n + row - p.row_starts[b];
    const int kvh = head / (p.q_heads / p.kv_heads);
    float q[V], o[V], m = -INFINITY, l = 0.0f;
    for (int i = 0; i < V; ++i) {
        q[i] = bf16_to_f32(p.q[row * p.q_stride + head * HD + lane * V + i]) * p.scale_log2;
        o[i] = 0.0f;
    }
    const long long limit = (long long)p.max_pages * p.page_tokens;
    const int end = len < n ? 0 : (int)min((long long)pos + 1, limit);
    for (int j = warp; j < end; j += kKv8SimpleWarps) {
        if (p.window > 0 && j >= p.sinks && j <= pos - p.window) continue;
        const int col = j / p.page_tokens, at = j - col * p.page_tokens;
        const int page = p.page_table[(long long)b * p.max_pages + col];
        if (page < 0 || page >= p.num_pages) continue;
        const long long h = (long long)page * p.kv_heads + kvh;
        const long long cell = (h * p.page_tokens + at) * HD + lane * V, block = h * (p.page_tokens / kKv8Block) + at / kKv8Block;
        float s = 0.0f, v[V];
        for (int i = 0; i < V; i += 2) {
            float f[4];
            unpack_e4m3x4(*reinterpret_cast<const uint16_t *>(p.k_codes + cell + i), f);
            s += q[i] * f[0] + q[i + 1] * f[1];
            unpack_e4m3x4(*reinterpret_cast<const uint16_t *>(p.v_codes + cell + i), f);
            v[i] = f[0] * p.v_scales[block];
            v[i + 1] = f[1] * p.v_scales[block];
        }
        s = warp_sum(s) * p.k_scales[block];
        const float to = fmaxf(m, s);
        const float f = exp2f(m - to), e = exp2f(s - to);
        m = to;
        l = l * f + e;
        for (int i = 0; i < V; ++i) o[i] = o[i] * f + e * v[i];
    }
    for (int i = 0; i < V; ++i) part_s[warp][lane * V + i] = o[i];
    if (lane == 0) {
        part_s[warp][HD] = m;
        part_s[warp][HD + 1] = l;
    }
    __syncthreads();
    if (warp != 0) return;
    float top = -INFINITY, sum = 0.0f;
    for (int w = 0; w < kKv8SimpleWarps; ++w) top = fmaxf(top, part_s[w][HD]);
    for (int i = 0; i < V; ++i) o[i] = 0.0f;
    for (int w = 0; w < kKv8SimpleWarps; ++w) {
        const float f = part_s[w][HD] == -INFINITY ? 0.0f : exp2f(part_s[w][HD] - top);
        sum += f * part_s[w][HD + 1];
        for (int i = 0; i < V; ++i) o[i] += f * part_s[w][lane * V + i];
    }
    for (int i = 0; i < V; ++i)
        p.out[((long long)row * p.q_heads + head) * HD + lane * V + i] = f32_to_bf16_rne(sum == 0.0f ? 0.0f : o[i] / sum);
}

}  // namespace cheetah
