// Block tables and slot maps of a step, from request lengths.
//
// Three running sums over the sequences (rows, pages) and then one cell per
// row: seq b's rows start at the exclusive sum of new_tokens, its new pages at
// the exclusive sum of need_b = ceil((c_b + n_b) / P) - ceil(c_b / P) in the
// free list, and row i of b is token c_b + i, in page (c_b + i) / P of b. The
// work is a few bytes per row, so a launch is bound by its latency: every CTA
// computes the sums of all sequences itself (at most 16384 of them, from L2)
// instead of waiting for another launch, then fills its share of the rows.
#pragma once

#include "common.cuh"

namespace cheetah {

constexpr int kSlotThreads = 512;
constexpr int kSlotWarps = kSlotThreads / kWarp;
constexpr int kSlotMaxBatch = 16384;

struct PageSlotParams {
    const int32_t *cached, *new_tokens, *free_pages, *free_count;
    int free_capacity;
    int batch;
    int32_t *page_table;
    int max_pages;
    int num_pages;
    int page_tokens;
    int max_tokens;
    int32_t *row_starts, *seq_lens, *positions, *seq_ids, *slots, *counts;
};

// Inclusive sum over the block; every thread also gets the block's total.
__device__ __forceinline__ long long block_scan(long long v, long long *warp_sums, long long &total) {
    const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
#pragma unroll
    for (int o = 1; o < kWarp; o <<= 1) {
        const long long up = __shfl_up_sync(0xFFFFFFFFu, v, o);
        if (lane >= o) v += up;
    }
    if (lane == kWarp - 1) warp_sums[warp] = v;
    __syncthreads();
    long long w = lane < kSlotWarps ? warp_sums[lane] : 0;
#pragma unroll
    for (int o = 1; o < kWarp; o <<= 1) {
        const long long up = __shfl_up_sync(0xFFFFFFFFu, w, o);
        if (lane >= o) w += up;
    }
    total = __shfl_sync(0xFFFFFFFFu, w, kSlotWarps - 1);
    const long long before = __shfl_sync(0xFFFFFFFFu, w, max(warp - 1, 0));
    __syncthreads();
    return warp > 0 ? v + before : v;
}

__global__ void __launch_bounds__(kSlotThreads) page_slots_kernel(const PageSlotParams p) {
    // Per sequence: end of its rows, free-list index minus its first new
    // page's table column, and that column (-1: refused).
    extern __shared__ int32_t slot_smem[];
    __shared__ long long warp_sums[kSlotWarps];
    int32_t *row_end = slot_smem, *free_base = row_end + p.batch, *first_new = free_base + p.batch;
    const long long capacity = (long long)p.max_pages * p.page_tokens;
    const int P = p.page_tokens;
    pdl_wait();
    pdl_launch_dependents();
    const int free_count = min(max(p.free_count[0], 0), p.free_capacity);

    long long rows_before = 0, pages_before = 0, pages_taken = 0;
    long long refused = 0;
    for (int b0 = 0; b0 < p.batch; b0 += kSlotThreads) {
        const int b = b0 + threadIdx.x;
        const bool real = b < p.batch;
        const long long c = real ? p.cached[b] : 0;
        long long n = real ? p.new_tokens[b] : 0;
        bool ok = c >= 0 && n >= 0 && c + n <= capacity;
        if (!ok) n = 0;
        long long total;
        const long long end = rows_before + block_scan(n, warp_sums, total);
        rows_before += total;
        ok = ok && end <= p.max_tokens;
        const long long have = ok ? (c + P - 1) / P : 0;
        const long long need = ok ? (c + n + P - 1) / P - have : 0;
        const long long page_end = pages_before + block_scan(need, warp_sums, total);
        pages_before += total;
        const bool got = ok && (need == 0 || page_end <= free_count);
        block_scan(got ? need : 0, warp_sums, total);
        pages_taken += total;
        block_scan(real && !got ? 1 : 0, warp_sums, total);
        refused += total;
        if (real) {
            row_end[b] = (int)min(end, (long long)p.max_tokens);
            free_base[b] = got ? (int)(page_end - need - have) : 0;
            first_new[b] = got ? (int)have : -1;
            if (blockIdx.x == 0) {
                p.row_starts[b + 1] = row_end[b];
                p.seq_lens[b] = got ? (int)(c + n) : 0;
            }
        }
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        p.row_starts[0] = 0;
        p.counts[0] = (int)min(rows_before, 0x7FFFFFFFll);
        p.counts[1] = (int)pages_taken;
        p.counts[2] = (int)refused;
    }
    __syncthreads();

    // Rows: sequence by binary search of the row ends, page from the free list
    // or from the part of the table that this launch leaves alone.
    const int live_rows = p.batch > 0 ? row_end[p.batch - 1] : 0;
    for (long long t = (long long)blockIdx.x * kSlotThreads + threadIdx.x; t < p.max_tokens;
         t += (long long)gridDim.x * kSlotThreads) {
        int pos = -1, seq = -1, slot = -1;
        if (t < live_rows) {
            int lo = 0, hi = p.batch - 1;
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (row_end[mid] > t) hi = mid;
                else lo = mid + 1;
            }
            seq = lo;
            const int fresh = first_new[lo];
            if (fresh >= 0) {
                pos = p.cached[lo] + (int)(t - (lo > 0 ? row_end[lo - 1] : 0));
                const int col = pos / P;
                const int page = col >= fresh ? p.free_pages[free_base[lo] + col]
                                              : p.page_table[(long long)lo * p.max_pages + col];
                if (page >= 0 && page < p.num_pages) slot = page * P + pos % P;
            }
        }
        p.positions[t] = pos;
        p.seq_ids[t] = seq;
        p.slots[t] = slot;
    }
    // Table entries of the new pages, a warp per sequence.
    const int lane = threadIdx.x % kWarp;
    for (int b = blockIdx.x * kSlotWarps + threadIdx.x / kWarp; b < p.batch; b += gridDim.x * kSlotWarps) {
        const int fresh = first_new[b];
        if (fresh < 0) continue;
        const int rows = row_end[b] - (b > 0 ? row_end[b - 1] : 0);
        const int last = (int)(((long long)p.cached[b] + rows + P - 1) / P);
        for (int col = fresh + lane; col < last; col += kWarp) {
            p.page_table[(long long)b * p.max_pages + col] = p.free_pages[free_base[b] + col];
        }
    }
}

}  // namespace cheetah
