// Log probability of a given token, its rank, the entropy and the likeliest
// tokens of each row of logits.
//
//   S = sum exp(x - m),  lse = m + log S,  log p_t = x_t - lse
//   H = log S + sum (m - x) exp(x - m) / S   (both terms >= 0: no cancellation)
//
// One CTA per row: a pass for the maximum, a pass for the sums, a pass per
// alternative.
#pragma once

#include "common.cuh"

namespace cheetah {

constexpr int kLpThreads = 512;
constexpr int kLpMaxTop = 32;

struct LogprobParams {
    const void *logits;
    long long row_stride;
    int rows, vocab;
    const int32_t *tokens;
    int top;
    float *logprob;
    int32_t *rank;
    float *entropy;
    int32_t *top_ids;
    float *top_logprobs;
};

template <typename T>
__device__ __forceinline__ float logit_at(const void *row, int i) {
    if constexpr (sizeof(T) == 2) return bf16_to_f32(static_cast<const uint16_t *>(row)[i]);
    else return static_cast<const float *>(row)[i];
}

// Order of the alternatives: larger value first, then the lower id, as one
// integer key (larger is better; 0 is none).
__device__ __forceinline__ unsigned long long top_key(float value, int id) {
    if (value == 0.0f) value = 0.0f;  // -0 and +0 are equal logits
    return ((unsigned long long)total_order_key(value) << 32) | (uint32_t)~id;
}
__device__ __forceinline__ float top_key_value(unsigned long long key) {
    const uint32_t k = (uint32_t)(key >> 32);
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

template <typename V, typename F>
__device__ __forceinline__ V block_reduce(V v, V *scratch, F f) {
    const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    __syncthreads();
    if (lane == 0) scratch[warp] = v;
    __syncthreads();
    V r = scratch[0];
    for (int w = 1; w < kLpThreads / kWarp; ++w) r = f(r, scratch[w]);
    return r;
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads) token_logprobs_kernel(const LogprobParams p) {
    __shared__ float f_scratch[kLpThreads / kWarp];
    __shared__ int i_scratch[kLpThreads / kWarp];
    __shared__ unsigned long long k_scratch[kLpThreads / kWarp];
    pdl_wait();
    pdl_launch_dependents();
    const int r = blockIdx.x;
    const void *row = static_cast<const T *>(p.logits) + r * p.row_stride;
    float m = -INFINITY;
    int bad = 0;
    for (int i = threadIdx.x; i < p.vocab; i += kLpThreads) {
        const float x = logit_at<T>(row, i);
        bad |= !(x < INFINITY);
        m = fmaxf(m, x);
    }
    m = block_reduce(m, f_scratch, [](float a, float b) { return fmaxf(a, b); });
    bad = block_reduce(bad, i_scratch, [](int a, int b) { return a | b; });
    bad |= m == -INFINITY;
    const int token = p.tokens[r];
    const bool known = token >= 0 && token < p.vocab;
    const float chosen = known && !bad ? logit_at<T>(row, token) : __int_as_float(0x7FC00000);
    float s = 0.0f, gap = 0.0f;
    int above = 0;
    for (int i = threadIdx.x; i < p.vocab; i += kLpThreads) {
        const float x = logit_at<T>(row, i);
        const float e = expf(x - m);
        s += e;
        gap += e > 0.0f ? (m - x) * e : 0.0f;
        above += x > chosen;
    }
    s = block_reduce(s, f_scratch, [](float a, float b) { return a + b; });
    gap = block_reduce(gap, f_scratch, [](float a, float b) { return a + b; });
    above = block_reduce(above, i_scratch, [](int a, int b) { return a + b; });
    const float nan = __int_as_float(0x7FC00000);
    const float log_s = logf(s);
    if (threadIdx.x == 0) {
        p.logprob[r] = bad || !known ? nan : (chosen - m) - log_s;
        if (p.rank) p.rank[r] = bad || !known ? 0 : 1 + above;
        if (p.entropy) p.entropy[r] = bad ? nan : log_s + gap / s;
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < p.top; ++k) {
        unsigned long long best = 0ull;
        if (!bad) {
            for (int i = threadIdx.x; i < p.vocab; i += kLpThreads) {
                const unsigned long long key = top_key(logit_at<T>(row, i), i);
                if (key < last && key > best) best = key;
            }
        }
        best = block_reduce(best, k_scratch, [](unsigned long long a, unsigned long long b) { return a > b ? a : b; });
        last = best;
        if (threadIdx.x == 0) {
            p.top_ids[(long long)r * p.top + k] = bad ? -1 : (int)~(uint32_t)best;
            p.top_logprobs[(long long)r * p.top + k] = bad ? nan : (top_key_value(best) - m) - log_s;
        }
    }
}

}  // namespace cheetah
