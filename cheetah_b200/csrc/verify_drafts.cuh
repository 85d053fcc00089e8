// Which drafted tokens a target keeps, and the token drawn behind them.
//
// Row r's draft x is kept while u q(x) < p(x); the next token is drawn from w =
// max(p - q, 0) at the first row that drops one, from w = p at a sequence's last
// row: the first v with w_0 + .. + w_v > u' W, W the sum of w.
//
// A cluster of CTAs per sequence. Each CTA finds the row for itself (a handful of
// gathered probabilities), sums its share of the row's weights in one pass, chunk by
// chunk, and learns the others' sums through distributed shared memory; the CTA
// whose share holds the token goes over the one chunk that does once more. So one
// row of p, and of q where a draft was dropped, is read, once.
//
// All sums and comparisons are f64: products of two f32 are exact there and
// differences nearly, and a running sum over 10^5 weights in f32 would move the
// borders between tokens by more than many of them are wide. A sum's order is
// fixed by the launch's shape.
//
// A short call is a chain of dependent reads (the starts, the tokens, their
// probabilities, the row, the sums' exchange, one chunk again): 7.8 us for one
// sequence of 5 rows over 151936 tokens, 7.5 us for 8. With many sequences it is
// bytes, of reads whose latency the lanes must cover: 96 sequences over 152064
// tokens, 58 MB of p and up to as much of q, take 23.3 us. Four vectors of each row
// in flight per lane beat two (33.8 us) and eight (29.3 us, whose registers leave
// two CTAs an SM).
#pragma once

#include <cooperative_groups.h>

#include "common.cuh"

namespace cheetah {

constexpr int kVdThreads = 256;
constexpr int kVdWarps = kVdThreads / kWarp;
constexpr int kVdMaxCluster = 16;
constexpr int kVdMaxChunks = 1024;  // of a CTA
constexpr int kVdLoads = 4;         // vectors of p (and of q) in flight per lane
constexpr int kVdResident = 3;      // CTAs of an SM that run at once

struct VerifyDraftsParams {
    const float *target, *draft;
    long long target_stride, draft_stride;
    int rows, vocab;
    const int32_t *tokens, *row_starts;
    int batch, parts;
    int chunk_vecs;   // vectors of 4 weights in a chunk, a multiple of kVdThreads
    const float *accept_u, *sample_u;
    int32_t *accepted, *out_tokens;
};

// Probability as f64: NaN and negative ones count as 0.
__device__ __forceinline__ double vd_prob(float x) { return x > 0.0f ? (double)x : 0.0; }

// The weights of one row: vectors of 4 from the 16-byte boundary at or before
// its first element on.
struct VdRow {
    const float *p, *q;   // q: nullptr where only p counts
    int vocab, shift;     // element 0 is number `shift` of vector 0
    bool same;            // q's vectors are aligned as p's
    int zero;             // a token of weight 0 (a certain draft that was dropped), or -1

    __device__ __forceinline__ void load(long long vec, float4 &a, float4 &b) const {
        const long long e = vec * 4 - shift;
        a = b = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (e >= 0 && e + 4 <= vocab) {
            a = __ldcs(reinterpret_cast<const float4 *>(p + e));
            if (q != nullptr) {
                if (same) b = __ldcs(reinterpret_cast<const float4 *>(q + e));
                else b = make_float4(q[e], q[e + 1], q[e + 2], q[e + 3]);
            }
        } else {
            float x[4] = {0.0f, 0.0f, 0.0f, 0.0f}, y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (e + i < 0 || e + i >= vocab) continue;
                x[i] = p[e + i];
                if (q != nullptr) y[i] = q[e + i];
            }
            a = make_float4(x[0], x[1], x[2], x[3]);
            b = make_float4(y[0], y[1], y[2], y[3]);
        }
    }
    __device__ __forceinline__ void weights(long long vec, const float4 &a, const float4 &b, double (&w)[4]) const {
        const float x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = vd_prob(x[i]);
            if (q != nullptr) w[i] = fmax(w[i] - vd_prob(y[i]), 0.0);
        }
        if (zero >= 0) {
            const long long at = zero + shift - vec * 4;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (at == i) w[i] = 0.0;
            }
        }
    }
};

__device__ __forceinline__ double vd_warp_sum(double v) {
#pragma unroll
    for (int o = kWarp / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}
// Sum of the lanes up to and including this one.
__device__ __forceinline__ double vd_warp_scan(double v) {
    const int lane = threadIdx.x % kWarp;
#pragma unroll
    for (int o = 1; o < kWarp; o <<= 1) {
        const double up = __shfl_up_sync(0xFFFFFFFFu, v, o);
        if (lane >= o) v += up;
    }
    return v;
}

__global__ void __launch_bounds__(kVdThreads, kVdResident) verify_drafts_kernel(const VerifyDraftsParams p) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    __shared__ double chunk_sum[kVdMaxChunks];
    __shared__ double part_sum[2][kVdMaxCluster];  // of every CTA; one array per pass
    __shared__ double warp_sum_s[kVdWarps];
    __shared__ int chosen, fallback;
    const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
    const int rank = (int)(blockIdx.x % p.parts), b = (int)(blockIdx.x / p.parts);
    pdl_wait();
    pdl_launch_dependents();
    const int r0 = min(max(p.row_starts[b], 0), p.rows), r1 = min(max(p.row_starts[b + 1], r0), p.rows);
    const int last = r1 - 1;
    if (last < r0) {  // (the whole cluster)
        if (rank == 0 && threadIdx.x == 0) p.accepted[b] = -1;
        return;
    }
    cluster.barrier_arrive();  // waited for before the first write into another CTA
    // The first row whose draft is not kept, or the last. Every warp looks.
    int stop = last;
    for (int r = r0; r < last; r += kWarp) {
        bool kept = true;
        if (r + lane < last) {
            const int x = p.tokens[r + lane + 1];
            kept = false;
            if (x >= 0 && x < p.vocab) {
                const double px = vd_prob(p.target[(r + lane) * p.target_stride + x]);
                const double qx = p.draft ? vd_prob(p.draft[(r + lane) * p.draft_stride + x]) : 1.0;
                kept = (double)p.accept_u[r + lane] * qx < px;
            }
        }
        const uint32_t dropped = __ballot_sync(0xFFFFFFFFu, !kept);
        if (dropped) {
            stop = r + __ffs(dropped) - 1;
            break;
        }
    }
    if (rank == 0) {
        if (threadIdx.x == 0) p.accepted[b] = stop - r0;
        for (int r = r0 + (int)threadIdx.x; r < r1; r += kVdThreads) {
            if (r != stop) p.out_tokens[r] = r < stop ? p.tokens[r + 1] : -1;
        }
    }
    const double u = (double)p.sample_u[b];
    VdRow row;
    row.p = p.target + stop * p.target_stride;
    row.q = nullptr;
    row.vocab = p.vocab;
    row.shift = (int)((uintptr_t)row.p >> 2 & 3);
    row.same = true;
    row.zero = -1;
    if (stop < last) {
        if (p.draft) {
            row.q = p.draft + stop * p.draft_stride;
            row.same = (((uintptr_t)row.q ^ (uintptr_t)row.p) & 15) == 0;
        } else {
            row.zero = p.tokens[stop + 1];
        }
    }
    const long long vecs = ((long long)p.vocab + row.shift + 3) / 4;
    const long long chunks = (vecs + p.chunk_vecs - 1) / p.chunk_vecs;
    const long long c0 = chunks * rank / p.parts, c1 = chunks * (rank + 1) / p.parts;
    const int own = (int)(c1 - c0);

    // Pass 0 with the row's weights; pass 1 with p alone, where those are all 0.
    double total = 0.0, before = 0.0;
    int used = 0;
    for (int pass = 0; pass < 2; ++pass) {
        for (int c = warp; c < own; c += kVdWarps) {
            const long long v0 = (c0 + c) * p.chunk_vecs;
            double sum = 0.0;
            for (int v = lane; v < p.chunk_vecs; v += kWarp * kVdLoads) {
                float4 a[kVdLoads], d[kVdLoads];
#pragma unroll
                for (int i = 0; i < kVdLoads; ++i) row.load(v0 + v + i * kWarp, a[i], d[i]);
#pragma unroll
                for (int i = 0; i < kVdLoads; ++i) {
                    double w[4];
                    row.weights(v0 + v + i * kWarp, a[i], d[i], w);
                    sum += (w[0] + w[1]) + (w[2] + w[3]);
                }
            }
            sum = vd_warp_sum(sum);
            if (lane == 0) chunk_sum[c] = sum;
        }
        __syncthreads();
        if (pass == 0) cluster.barrier_wait();
        if (warp == 0) {
            double sum = 0.0;
            for (int c = lane; c < own; c += kWarp) sum += chunk_sum[c];
            sum = vd_warp_sum(sum);
            if (lane < p.parts) *cluster.map_shared_rank(&part_sum[pass][rank], lane) = sum;
        }
        cluster.sync();
        total = 0.0;
        used = pass;
        for (int i = 0; i < p.parts; ++i) {
            if (i == rank) before = total;
            total += part_sum[pass][i];
        }
        if (total > 0.0 || (row.q == nullptr && row.zero < 0)) break;
        row.q = nullptr;
        row.zero = -1;
    }
    if (!(total > 0.0 && total < INFINITY)) {
        if (rank == 0 && threadIdx.x == 0) p.out_tokens[stop] = -1;
        return;
    }
    // The part that holds the token: the first whose end passes u W, or else the
    // last of positive weight. Every CTA has the same sums in the same order.
    const double target = u * total;
    int owner = -1;
    double end = 0.0;
    for (int i = 0; i < p.parts; ++i) {
        const double s = part_sum[used][i];
        end += s;
        if (s > 0.0) owner = i;
        if (end > target) break;
    }
    if (owner != rank) return;
    // Within the part: the chunk, by the same rule.
    if (warp == 0) {
        double run = before;
        int found = -1, some = -1;
        double found_before = 0.0, some_before = 0.0;
        for (int c = 0; c < own && found < 0; c += kWarp) {
            const double s = c + lane < own ? chunk_sum[c + lane] : 0.0;
            const double upto = run + vd_warp_scan(s);
            const uint32_t positive = __ballot_sync(0xFFFFFFFFu, s > 0.0);
            const uint32_t past = __ballot_sync(0xFFFFFFFFu, s > 0.0 && upto > target);
            const uint32_t pick = past ? past & -past : (positive ? 1u << (31 - __clz(positive)) : 0u);
            if (pick) {
                const int at = __ffs(pick) - 1;
                const double start = __shfl_sync(0xFFFFFFFFu, upto - s, at);
                some = c + at;
                some_before = start;
                if (past) {
                    found = some;
                    found_before = start;
                }
            }
            run = __shfl_sync(0xFFFFFFFFu, upto, kWarp - 1);
        }
        if (lane == 0) {
            chosen = found >= 0 ? found : some;
            warp_sum_s[0] = found >= 0 ? found_before : some_before;
            fallback = -1;
        }
    }
    __syncthreads();
    const int chunk = chosen;
    double run = warp_sum_s[0];
    __syncthreads();
    if (chunk < 0) return;
    // The token: the block scans the chunk, kVdThreads vectors at a time.
    for (int v = 0; v < p.chunk_vecs; v += kVdThreads) {
        const long long vec = (c0 + chunk) * (long long)p.chunk_vecs + v + threadIdx.x;
        float4 a, d;
        double w[4];
        row.load(vec, a, d);
        row.weights(vec, a, d, w);
        const double sum = (w[0] + w[1]) + (w[2] + w[3]);
        const double upto = vd_warp_scan(sum);
        if (lane == kWarp - 1) warp_sum_s[warp] = upto;
        if (threadIdx.x == 0) chosen = kVdThreads;
        __syncthreads();
        double base = run;
        for (int i = 0; i < kVdWarps; ++i) {
            if (i < warp) base += warp_sum_s[i];
            run += warp_sum_s[i];
        }
        double at = base + (upto - sum);
        int hit = -1, some = -1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            at += w[i];
            if (w[i] > 0.0) {
                some = i;
                if (hit < 0 && at > target) hit = i;
            }
        }
        if (hit >= 0) atomicMin(&chosen, (int)threadIdx.x);
        if (some >= 0) atomicMax(&fallback, (int)(vec * 4 - row.shift + some));
        __syncthreads();
        const int winner = chosen;
        if (winner < kVdThreads) {
            if ((int)threadIdx.x == winner) p.out_tokens[stop] = (int)(vec * 4 - row.shift + hit);
            return;
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) p.out_tokens[stop] = fallback;
}

}  // namespace cheetah
