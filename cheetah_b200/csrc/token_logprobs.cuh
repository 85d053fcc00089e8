// Log probability of a given token, its rank, the entropy and the likeliest
// tokens of each row of logits, in one pass over the row.
//
//   S = sum exp(x - m),  lse = m + log S,  log p_t = x_t - lse
//   H = log S + sum (m - x) exp(x - m) / S   (both terms >= 0: no cancellation)
//
// with m the row's largest logit. A thread sums about a reference of its own, at
// most kLpHeadroom below the largest that it has met, and goes over to that one
// at the end: moving m to m' multiplies S by f = exp(m - m') and G = sum (x - m)
// exp(x - m) becomes f (G + (m - m') S).
//
// Bound by memory where rows are many, by latency where they are few: a row
// is split over a cluster of 1..16 CTAs that join their results in the first
// one's shared memory, so a call is one launch and needs no workspace.
//
// One f32 row of 151936 with 5 alternatives takes 8.7 us (16 CTAs; latency),
// 2048 such rows with one 214 .. 218 us (5.7 .. 5.8 TB/s), 500 bf16 rows of
// 152064 38 us without alternatives and 55 us (2.8 TB/s) with twenty: there the
// operations per logit bound it (about 8, and a logit is 2 bytes), the sorts,
// and that 500 rows leave a sixth of the SMs' places empty.
//
// Alternatives. Each (warp, j) pair owns a contiguous run of 512-byte pieces
// of the CTA's part and one iteration reads the next piece of every run, so
// the first iteration samples the whole part. The `top`-th best of the
// threads' first maxima is a lower bound of the part's `top`-th best value;
// elements at or above it go to a buffer, from which each warp sorts its share
// in registers and the warps' lists are merged pairwise; done once after a
// quarter of the part, this gives a closer bound for the rest (about 13 * top
// candidates in all instead of 40 * top). Where they do not fit (an
// adversarial order), the exact `top`-th key is found by a radix selection over
// the part instead, in 8 more passes.
#pragma once

#include <cooperative_groups.h>

#include "common.cuh"

namespace cheetah {

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / kWarp;
constexpr int kLpMaxTop = 32;
constexpr int kLpMaxCluster = 16;
constexpr int kLpLoads = 4;        // 16-byte loads in flight per thread
constexpr int kLpBuffer = 1024;    // candidates of a CTA
constexpr int kLpAhead = 4;        // iterations asked for ahead of a sort
// From this many alternatives on a second bound pays for its sort: 500 bf16
// rows of 152064 with twenty take 88 us without it, 57 with one after an eighth
// and 54 after a quarter; 2048 f32 rows with one alternative 217 and 220.
constexpr int kLpRefineTop = 4;
constexpr float kLpLog2e = 1.4426950408889634f;
constexpr float kLpFloor = -1.0e4f;  // 2^floor is 0; keeps t * 0 finite
// Logits this far above a thread's reference move it: a sum about a reference
// that lies t log2 units below the largest logit is off by t 2^-24. 500 bf16 rows
// with twenty alternatives take 55.3 us with 1, 55.0 with 2 or 8.
constexpr float kLpHeadroom = 1.0f;
constexpr float kLpFused = 1048576.0f;  // largest logit whose log2(e) multiple rounds to within 1/8

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

using TopKey = unsigned long long;

// Order of the alternatives: larger value first, then the lower id, as one
// integer key (larger is better; 0 is none).
__device__ __forceinline__ TopKey top_key(float value, int id) {
    if (value == 0.0f) value = 0.0f;  // -0 and +0 are equal logits
    return ((TopKey)total_order_key(value) << 32) | (uint32_t)~id;
}
__device__ __forceinline__ float total_order_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k); }
__device__ __forceinline__ float top_key_value(TopKey key) { return total_order_value((uint32_t)(key >> 32)); }

// max(a, b), NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Sums of a row part about a logit m, in log2 units: s = sum 2^t, gap = sum t
// 2^t with t = log2(e) (x - m). A NaN or +inf logit makes s NaN; a part
// without a logit above -inf has s = 0.
struct RowSums {
    float m, s, gap;

    __device__ __forceinline__ void init() {
        m = -3.402823466e38f;
        s = gap = 0.0f;
    }
    __device__ __forceinline__ void raise(float to) {
        const float t = max_nan((m - to) * kLpLog2e, kLpFloor);
        const float f = fast_exp2(t);
        gap = f * fmaf(t, s, gap);
        s *= f;
        m = to;
    }
    // Any logit: every case is in order, for a few more operations.
    __device__ __forceinline__ void add(float x) {
        if (x > m) raise(x);
        const float t = max_nan((x - m) * kLpLog2e, kLpFloor);
        const float e = fast_exp2(t);
        s += e;
        gap = fmaf(t, e, gap);
    }
    __device__ __forceinline__ void join(const RowSums &o) {
        RowSums other = o;
        const float to = fmaxf(m, o.m);
        raise(to);
        other.raise(to);
        s += other.s;
        gap += other.gap;
    }
};

// The same sums as the stream over the row takes them: about a whole number r
// of log2 units, exact in f32, so t = log2(e) x - r is one fused operation
// with one rounding. r begins at the largest logit of the warp's first loads and
// moves only when a logit lies kLpHeadroom above it. A logit of -inf adds 0 to s
// but makes gap NaN, and logits beyond kLpFused have no such r; then `blurred` is
// set and the part is summed once more, by RowSums::add().
struct StreamSums {
    float r, s, gap, limit, peak;
    bool blurred;

    __device__ __forceinline__ void init() {
        r = s = gap = 0.0f;
        limit = peak = -INFINITY;
        blurred = false;
    }
    __device__ __forceinline__ void move(float to_m) {
        const float to = rintf(to_m * kLpLog2e);
        const float shift = fmaxf(r - to, kLpFloor);
        const float f = s > 0.0f ? fast_exp2(shift) : 0.0f;
        gap = f * fmaf(shift, s, gap);
        s *= f;
        r = to;
        peak = fmaxf(peak, to_m);
        limit = to_m + kLpHeadroom;
        blurred |= !(fabsf(to_m) < kLpFused);
    }
    __device__ __forceinline__ void add(float x) {
        const float t = fmaf(x, kLpLog2e, -r);
        const float e = fast_exp2(t);
        s += e;
        gap = fmaf(t, e, gap);
    }
    // The sums about the largest logit that this thread has met. Its term is
    // divided by itself, so where it is the row's largest s is at least 1, and
    // no gap is positive: no probability comes out above 1, no entropy below 0.
    __device__ __forceinline__ RowSums about_peak() {
        RowSums o;
        o.init();
        if (peak > -INFINITY) {
            o.m = peak;
            const float t = fmaf(peak, kLpLog2e, -r);
            const float e = fast_exp2(t);
            o.s = s / e;
            o.gap = fminf(fmaf(-t, s, gap) / e, 0.0f);
        }
        blurred |= !(gap == gap);
        return o;
    }
};

// The larger of each half, as bf16.
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// 1 or 0 per half, and their sums.
__device__ __forceinline__ uint32_t gt_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("set.gt.bf16x2.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t add_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

template <typename T>
struct LogitVec {
    static constexpr int N = 16 / sizeof(T);
    static __device__ __forceinline__ void widen(const uint4 &raw, float *v) {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 2) {
                v[2 * i] = bf16_lo(w[i]);
                v[2 * i + 1] = bf16_hi(w[i]);
            } else {
                v[i] = __uint_as_float(w[i]);
            }
        }
    }
    // The largest value of a vector (NaN left out); v: the vector widened.
    static __device__ __forceinline__ float largest(const uint4 &raw, const float *v) {
        if constexpr (sizeof(T) == 2) {
            const uint32_t m = max_bf16x2(max_bf16x2(raw.x, raw.y), max_bf16x2(raw.z, raw.w));
            return fmaxf(bf16_lo(m), bf16_hi(m));
        } else {
            return fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
        }
    }
    // Value i of a vector.
    static __device__ __forceinline__ float pick(const uint4 &raw, int i) {
        const int word = i * (int)sizeof(T) / 4;
        const uint32_t w = word < 2 ? (word == 0 ? raw.x : raw.y) : (word == 2 ? raw.z : raw.w);
        if constexpr (sizeof(T) == 2) return (i & 1) ? bf16_hi(w) : bf16_lo(w);
        else return __uint_as_float(w);
    }
    // How many values of a vector are above `than`.
    static __device__ __forceinline__ int above(const uint4 &raw, const float *v, float than) {
        if constexpr (sizeof(T) == 2) {
            uint32_t limit;
            asm("cvt.rn.bf16x2.f32 %0, %1, %1;" : "=r"(limit) : "f"(than));  // a bf16 logit, or +inf: exact
            const uint32_t n = add_bf16x2(add_bf16x2(gt_bf16x2(raw.x, limit), gt_bf16x2(raw.y, limit)),
                                          add_bf16x2(gt_bf16x2(raw.z, limit), gt_bf16x2(raw.w, limit)));
            return (int)(bf16_lo(n) + bf16_hi(n));
        } else {
            return (v[0] > than) + (v[1] > than) + (v[2] > than) + (v[3] > than);
        }
    }
    static __device__ __forceinline__ float one(const T *row, long long i) {
        if constexpr (sizeof(T) == 2) return bf16_to_f32(reinterpret_cast<const uint16_t *>(row)[i]);
        else return row[i];
    }
};

struct LogprobShared {
    TopKey buffer[kLpBuffer];
    TopKey lists[kLpWarps][kWarp];            // sorted lists on their way to one
    TopKey joined[kLpMaxCluster][kWarp];      // first CTA: every part's best
    float4 part[kLpMaxCluster];               // first CTA: m, s, gap, rank count bits
    float4 warp_part[kLpWarps];
    TopKey prefix;
    int histogram[256];
    int count, need;
};
static_assert(kLpMaxTop <= kWarp && kLpMaxCluster <= 2 * kLpWarps, "a list is one key per lane, two are merged by a warp");

// Bitonic steps over the warp's lanes; the best key ends in lane 0.
__device__ __forceinline__ TopKey lane_exchange(TopKey k, int stride, bool best_low) {
    const TopKey other = __shfl_xor_sync(0xFFFFFFFFu, k, stride);
    const bool low = (threadIdx.x & stride) == 0;
    return (low == best_low) == (k > other) ? k : other;
}
__device__ __forceinline__ TopKey warp_sort(TopKey k) {
#pragma unroll
    for (int size = 2; size <= kWarp; size <<= 1) {
#pragma unroll
        for (int stride = size / 2; stride > 0; stride >>= 1) k = lane_exchange(k, stride, (threadIdx.x & size & (kWarp - 1)) == 0);
    }
    return k;
}
// The best 32 of two sorted lists, sorted.
__device__ __forceinline__ TopKey warp_merge(TopKey a, TopKey b) {
    const TopKey back = __shfl_sync(0xFFFFFFFFu, b, (kWarp - 1) - (threadIdx.x & (kWarp - 1)));
    TopKey k = a > back ? a : back;
#pragma unroll
    for (int stride = kWarp / 2; stride > 0; stride >>= 1) k = lane_exchange(k, stride, true);
    return k;
}
// Merges lists[0..n) (n a power of two) into lists[0]. Every thread of the
// block calls it, the lists' writers before a barrier of this function's.
__device__ __forceinline__ void merge_lists(TopKey (*lists)[kWarp], int n) {
    const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
    __syncthreads();
    for (int half = n / 2; half > 0; half >>= 1) {
        if (warp < half) lists[warp][lane] = warp_merge(lists[warp][lane], lists[warp + half][lane]);
        __syncthreads();
    }
}
// The best 32 of keys[0..n), sorted, to lists[0].
__device__ __forceinline__ void pick_best(const TopKey *keys, int n, TopKey (*lists)[kWarp]) {
    const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
    TopKey mine = 0ull;
    for (int i = warp * kWarp; i < n; i += kLpThreads) {
        const TopKey k = warp_sort(i + lane < n ? keys[i + lane] : 0ull);
        mine = i < kLpThreads ? k : warp_merge(mine, k);
    }
    lists[warp][lane] = mine;
    merge_lists(lists, kLpWarps);
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads, 4) token_logprobs_kernel(const LogprobParams p) {
    namespace cg = cooperative_groups;
    using V = LogitVec<T>;
    constexpr int N = V::N;
    __shared__ LogprobShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int r = blockIdx.x / parts;
    const int tid = threadIdx.x, lane = tid % kWarp, warp = tid / kWarp;
    if (tid == 0) sh.count = 0;
    cluster.barrier_arrive();  // waited for before another CTA's shared memory is written
    pdl_wait();
    pdl_launch_dependents();
    const T *row = static_cast<const T *>(p.logits) + r * p.row_stride;
    // Elements before the first 16-byte boundary, whole vectors, the rest.
    const int head = min(p.vocab, (int)((16 - ((uintptr_t)row & 15)) & 15) / (int)sizeof(T));
    const int vecs = (p.vocab - head) / N;
    const int tail0 = head + vecs * N;
    const uint4 *vec = reinterpret_cast<const uint4 *>(row + head);
    const int v0 = (int)((long long)vecs * rank / parts), v1 = (int)((long long)vecs * (rank + 1) / parts);
    const int lines = (v1 - v0 + kWarp - 1) / kWarp;
    const int run = (lines + kLpWarps * kLpLoads - 1) / (kLpWarps * kLpLoads);
    // Vector of load j in iteration it (>= v1: none).
    auto vector_at = [&](int it, int j) -> int { return v0 + ((warp * kLpLoads + j) * run + it) * kWarp + lane; };
    // Asks L2 for the lines of the coming iterations, so that DRAM keeps busy
    // while the threads sort.
    auto ask_ahead = [&](int it) {
#pragma unroll 1
        for (int a = it; a < min(it + kLpAhead, run); ++a) {
#pragma unroll
            for (int j = 0; j < kLpLoads; ++j) {
                const int v = vector_at(a, j);
                if (v < v1 && lane % 8 == 0) asm volatile("prefetch.global.L2 [%0];" ::"l"(vec + v));
            }
        }
    };
    // The odd elements at the row's ends: one each for a few threads of the first CTA.
    int odd = -1;
    if (rank == 0) {
        if (tid < head) odd = tid;
        else if (tid - head < p.vocab - tail0) odd = tail0 + tid - head;
    }

    const int token = p.tokens[r];
    const bool known = token >= 0 && token < p.vocab;
    const float chosen = known ? V::one(row, token) : INFINITY;

    StreamSums stream;
    stream.init();
    int above = 0;
    float tau = INFINITY;
    TopKey tau_key = ~0ull;
    auto push = [&](float x, int id) {
        const TopKey key = top_key(x, id);
        if (key < tau_key) return;
        const int at = atomicAdd(&sh.count, 1);
        if (at < kLpBuffer) sh.buffer[at] = key;
    };
    auto consume = [&](const uint4 (&raw)[kLpLoads], int it) {
#pragma unroll
        for (int j = 0; j < kLpLoads; ++j) {
            const int v = vector_at(it, j);
            if (v >= v1) break;
            float x[N];
            V::widen(raw[j], x);
            const float mx = V::largest(raw[j], x);
            stream.peak = fmaxf(stream.peak, mx);
            if (mx > stream.limit) stream.move(mx);
#pragma unroll
            for (int i = 0; i < N; ++i) stream.add(x[i]);
            above += V::above(raw[j], x, chosen);
            if (mx >= tau) {
                uint32_t near = 0;
#pragma unroll
                for (int i = 0; i < N; ++i) near |= x[i] >= tau ? 1u << i : 0u;
#pragma unroll 1
                for (; near; near &= near - 1) {
                    const int i = __ffs(near) - 1;
                    push(V::pick(raw[j], i), head + v * N + i);
                }
            }
        }
    };
    auto load = [&](uint4 (&raw)[kLpLoads], int it) {
#pragma unroll
        for (int j = 0; j < kLpLoads; ++j) {
            const int v = vector_at(it, j);
            if (it < run && v < v1) raw[j] = __ldcs(vec + v);
        }
    };
    uint4 raw[kLpLoads];
    load(raw, 0);
    // The warp's sample sets its reference.
    float high = -INFINITY;
#pragma unroll
    for (int j = 0; j < kLpLoads; ++j) {
        if (run > 0 && vector_at(0, j) < v1) {
            float x[N];
            V::widen(raw[j], x);
            high = fmaxf(high, V::largest(raw[j], x));
        }
    }
    high = total_order_value(__reduce_max_sync(0xFFFFFFFFu, total_order_key(high)));
    if (high > -INFINITY) stream.move(high);
    if (p.top > 0) {
        ask_ahead(1);
        TopKey mine = odd >= 0 ? top_key(V::one(row, odd), odd) : 0ull;
#pragma unroll
        for (int j = 0; j < kLpLoads; ++j) {
            const int v = vector_at(0, j);
            if (run == 0 || v >= v1) break;
            float x[N];
            V::widen(raw[j], x);
            const float mx = V::largest(raw[j], x);
            int at = -1;
#pragma unroll
            for (int i = N - 1; i >= 0; --i) {
                if (x[i] == mx) at = i;
            }
            const TopKey key = at >= 0 ? top_key(mx, head + v * N + at) : 0ull;
            mine = key > mine ? key : mine;
        }
        sh.lists[warp][lane] = warp_sort(mine);
        merge_lists(sh.lists, kLpWarps);
        tau_key = sh.lists[0][p.top - 1];
        tau = tau_key ? top_key_value(tau_key) : -INFINITY;
    }
    auto stream_over = [&](int from, int to) {
        for (int it = from; it < to; ++it) {
            uint4 next[kLpLoads];
            load(next, it + 1);
            consume(raw, it);
#pragma unroll
            for (int j = 0; j < kLpLoads; ++j) raw[j] = next[j];
        }
    };
    int done = 0;
    if (p.top >= kLpRefineTop && run >= 4) {
        // The best of a quarter of the part: a closer bound for the rest.
        done = (run + 2) / 4;
        stream_over(0, done);
        ask_ahead(done + 1);
        __syncthreads();
        const int count = sh.count;
        if (count <= kLpBuffer) {
            pick_best(sh.buffer, count, sh.lists);
            if (tid < kWarp) sh.buffer[tid] = sh.lists[0][tid];
            if (tid == 0) sh.count = min(count, kWarp);
            const TopKey closer = sh.lists[0][p.top - 1];
            if (closer > tau_key) {
                tau_key = closer;
                tau = top_key_value(closer);
            }
        }
        __syncthreads();
    }
    stream_over(done, run);

    RowSums sums = stream.about_peak();
    if (__syncthreads_or(stream.blurred)) {
        sums.init();
        for (int id = head + v0 * N + tid; id < head + v1 * N; id += kLpThreads) sums.add(V::one(row, id));
    }
    if (odd >= 0) {
        const float x = V::one(row, odd);
        sums.add(x);
        above += x > chosen;
        if (p.top > 0 && x >= tau) push(x, odd);
    }

    // This part's sums, and its best keys.
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        RowSums other;
        other.m = __shfl_xor_sync(0xFFFFFFFFu, sums.m, o);
        other.s = __shfl_xor_sync(0xFFFFFFFFu, sums.s, o);
        other.gap = __shfl_xor_sync(0xFFFFFFFFu, sums.gap, o);
        sums.join(other);
        above += __shfl_xor_sync(0xFFFFFFFFu, above, o);
    }
    if (lane == 0) sh.warp_part[warp] = make_float4(sums.m, sums.s, sums.gap, __int_as_float(above));
    __syncthreads();
    if (p.top > 0) {
        if (sh.count <= kLpBuffer) {
            pick_best(sh.buffer, sh.count, sh.lists);
        } else {
            // The top-th key of this part, 8 bits at a time from the highest.
            auto for_each = [&](auto f) {
                for (int v = v0 + tid; v < v1; v += kLpThreads) {
                    float x[N];
                    V::widen(vec[v], x);
                    for (int i = 0; i < N; ++i) {
                        if (x[i] == x[i]) f(top_key(x[i], head + v * N + i));
                    }
                }
                if (odd >= 0) f(top_key(V::one(row, odd), odd));
            };
            if (tid == 0) {
                sh.prefix = 0ull;
                sh.need = p.top;
            }
            for (int shift = 56; shift >= 0; shift -= 8) {
                if (tid < 256) sh.histogram[tid] = 0;
                __syncthreads();
                const TopKey prefix = sh.prefix;
                for_each([&](TopKey k) {
                    if (shift == 56 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&sh.histogram[(k >> shift) & 255], 1);
                });
                __syncthreads();
                if (tid == 0) {
                    int need = sh.need, digit = 255;
                    while (digit > 0 && sh.histogram[digit] < need) need -= sh.histogram[digit--];
                    sh.need = need;
                    sh.prefix = prefix | ((TopKey)digit << shift);
                    sh.count = 0;
                }
                __syncthreads();
            }
            const TopKey last = sh.prefix;
            for_each([&](TopKey k) {
                if (k >= last) sh.buffer[atomicAdd(&sh.count, 1)] = k;
            });
            __syncthreads();
            pick_best(sh.buffer, min(sh.count, kLpBuffer), sh.lists);
        }
    }

    // Join the parts in the first CTA, which is running once all have arrived.
    cluster.barrier_wait();
    LogprobShared *first = cluster.map_shared_rank(&sh, 0);
    if (tid == 0) {
        RowSums all;
        all.init();
        int count = 0;
        for (int w = 0; w < kLpWarps; ++w) {
            const float4 q = sh.warp_part[w];
            RowSums other;
            other.m = q.x;
            other.s = q.y;
            other.gap = q.z;
            all.join(other);
            count += __float_as_int(q.w);
        }
        first->part[rank] = make_float4(all.m, all.s, all.gap, __int_as_float(count));
    }
    if (p.top > 0 && tid < kWarp) first->joined[rank][tid] = sh.lists[0][tid];
    cluster.sync();
    if (rank != 0) return;
    RowSums all;
    all.init();
    int count = 0;
    for (int w = 0; w < parts; ++w) {
        const float4 q = sh.part[w];
        RowSums other;
        other.m = q.x;
        other.s = q.y;
        other.gap = q.z;
        all.join(other);
        count += __float_as_int(q.w);
    }
    const bool bad = !(all.s > 0.0f);
    const float nan = __int_as_float(0x7FC00000);
    const float log_s = logf(all.s);
    if (tid == 0) {
        p.logprob[r] = bad || !known ? nan : (chosen - all.m) - log_s;
        if (p.rank) p.rank[r] = bad || !known ? 0 : 1 + count;
        if (p.entropy) p.entropy[r] = bad ? nan : log_s - 0.69314718056f * (all.gap / all.s);
    }
    if (p.top > 0) {
        merge_lists(sh.joined, parts);
        if (tid < p.top) {
            const TopKey key = sh.joined[0][tid];
            const long long at = (long long)r * p.top + tid;
            p.top_ids[at] = bad ? -1 : (int)~(uint32_t)key;
            p.top_logprobs[at] = bad ? nan : (top_key_value(key) - all.m) - log_s;
        }
    }
}

}  // namespace cheetah
