// Per-head RMSNorm of q and k, rotation at a given position, append of K and
// V at a given slot, in one pass over the fused projection rows.
//
//   y = x * (1/sqrt(mean(x^2) + eps) * w)        (heads with a norm weight)
//   (a, b) -> (a cos - b sin, b cos + a sin)      (pairs i, i + rotary/2)
//
// One warp per (row, head); f32 arithmetic, one rounding to the output type.
#pragma once

#include "common.cuh"

namespace cheetah {

struct QkNormRopeParams {
    const void *qkv;
    long long qkv_stride;
    const float *q_norm, *k_norm;
    float eps;
    const float *rope_cos, *rope_sin;
    int max_positions, rotary_dim;
    const int32_t *positions, *slots;
    int tokens, q_heads, kv_heads, head_dim;
    void *q_out, *k_pool, *v_pool;
    int num_pages, page_tokens;
};

template <typename T>
__device__ __forceinline__ float load_f32(const void *base, long long i) {
    if constexpr (sizeof(T) == 2) return bf16_to_f32(static_cast<const uint16_t *>(base)[i]);
    else return static_cast<const float *>(base)[i];
}
template <typename T>
__device__ __forceinline__ void store_f32(void *base, long long i, float v) {
    if constexpr (sizeof(T) == 2) static_cast<uint16_t *>(base)[i] = f32_to_bf16_rne(v);
    else static_cast<float *>(base)[i] = v;
}

template <typename TIN, typename TKV>
__global__ void __launch_bounds__(128) qk_norm_rope_rows_kernel(const QkNormRopeParams p) {
    const int heads = p.q_heads + 2 * p.kv_heads;
    const int lane = threadIdx.x % kWarp;
    const long long item = (long long)blockIdx.x * 4 + threadIdx.x / kWarp;
    pdl_wait();
    pdl_launch_dependents();
    if (item >= (long long)p.tokens * heads) return;
    const int t = (int)(item / heads), head = (int)(item % heads);
    const int pos = p.positions[t];
    if (pos < 0 || pos >= p.max_positions) return;
    const int hd = p.head_dim, half = p.rotary_dim / 2;
    const bool is_q = head < p.q_heads;
    const bool is_k = !is_q && head < p.q_heads + p.kv_heads;
    const float *w = is_q ? p.q_norm : (is_k ? p.k_norm : nullptr);
    const long long src = t * p.qkv_stride + (long long)head * hd;
    float inv = 1.0f;
    if (w) {
        float ss = 0.0f;
        for (int d = lane; d < hd; d += kWarp) {
            const float x = load_f32<TIN>(p.qkv, src + d);
            ss = fmaf(x, x, ss);
        }
        inv = 1.0f / sqrtf(warp_sum(ss) / (float)hd + p.eps);
    }
    long long dst;
    if (is_q) {
        dst = ((long long)t * p.q_heads + head) * hd;
    } else {
        const int slot = p.slots[t];
        if (slot < 0 || slot / p.page_tokens >= p.num_pages) return;
        const int kvh = is_k ? head - p.q_heads : head - p.q_heads - p.kv_heads;
        dst = (((long long)(slot / p.page_tokens) * p.kv_heads + kvh) * p.page_tokens + slot % p.page_tokens) * hd;
    }
    for (int d = lane; d < hd; d += kWarp) {
        float x = load_f32<TIN>(p.qkv, src + d);
        if (w) x *= inv * w[d];
        if ((is_q || is_k) && d < 2 * half) {
            const int i = d < half ? d : d - half;
            const int other = d < half ? d + half : d - half;
            float y = load_f32<TIN>(p.qkv, src + other);
            if (w) y *= inv * w[other];
            const float c = p.rope_cos[(long long)pos * half + i], s = p.rope_sin[(long long)pos * half + i];
            x = d < half ? x * c - y * s : x * c + y * s;
        }
        if (is_q) store_f32<TIN>(p.q_out, dst + d, x);
        else store_f32<TKV>(is_k ? p.k_pool : p.v_pool, dst + d, x);
    }
}

}  // namespace cheetah
