// Block tables and slot maps of a step, from request lengths.
//
// Three running sums over the sequences (rows, pages) and then one cell per
// row: seq b's rows start at the exclusive sum of new_tokens, its new pages at
// the exclusive sum of need_b = ceil((c_b + n_b) / P) - ceil(c_b / P) in the
// free list, and row i of b is token c_b + i, in page (c_b + i) / P of b. The
// work is a few bytes per row, so a launch is bound by its latency: every CTA
// computes the sums of all sequences itself (at most 16384 of them, from L2)
// instead of waiting for another launch, then fills its share of the rows.
// 64 sequences with 541 new rows take 4.1 us (one chain of dependent reads:
// lengths, sums, table, page), 256 sequences with a million rows 12.8 us
// (13.7 MB, 1.1 TB/s).
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

// VEC 4 needs 16-byte aligned per-row outputs.
template <int VEC>
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

    long long rows_before = 0, pages_before = 0, tally = 0;
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
        if (blockIdx.x == 0) {  // pages taken (< 2^31) and sequences refused (< 2^15) in one sum
            block_scan(((got ? need : 0) << 16) + (real && !got ? 1 : 0), warp_sums, total);
            tally += total;
        }
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
        p.counts[1] = (int)(tally >> 16);
        p.counts[2] = (int)(tally & 0xFFFF);
    }
    __syncthreads();

    // Rows, VEC at a time: the first one's sequence by binary search of the row
    // ends, the others' by stepping on; pages from the free list or from the
    // part of the table that this launch leaves alone.
    const int live_rows = row_end[p.batch - 1];
    for (long long t0 = ((long long)blockIdx.x * kSlotThreads + threadIdx.x) * VEC; t0 < p.max_tokens;
         t0 += (long long)gridDim.x * kSlotThreads * VEC) {
        int pos[VEC], seq[VEC], slot[VEC];
        int b = 0;
        if (t0 < live_rows) {
            int hi = p.batch - 1;
            while (b < hi) {
                const int mid = (b + hi) >> 1;
                if (row_end[mid] > t0) hi = mid;
                else b = mid + 1;
            }
        }
        int col_have = -1, page = -1;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const long long t = t0 + i;
            pos[i] = seq[i] = slot[i] = -1;
            if (t >= live_rows) continue;
            while (row_end[b] <= t) {
                ++b;
                col_have = -1;
            }
            seq[i] = b;
            const int fresh = first_new[b];
            if (fresh < 0) continue;
            pos[i] = p.cached[b] + (int)(t - (b > 0 ? row_end[b - 1] : 0));
            const int col = pos[i] / P;
            if (col != col_have) {
                col_have = col;
                page = col >= fresh ? p.free_pages[free_base[b] + col] : p.page_table[(long long)b * p.max_pages + col];
            }
            if (page >= 0 && page < p.num_pages) slot[i] = page * P + pos[i] - col * P;
        }
        if constexpr (VEC == 4) {
            if (t0 + VEC <= p.max_tokens) {
                *reinterpret_cast<int4 *>(p.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
                *reinterpret_cast<int4 *>(p.seq_ids + t0) = make_int4(seq[0], seq[1], seq[2], seq[3]);
                *reinterpret_cast<int4 *>(p.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
                continue;
            }
        }
        for (int i = 0; i < VEC && t0 + i < p.max_tokens; ++i) {
            p.positions[t0 + i] = pos[i];
            p.seq_ids[t0 + i] = seq[i];
            p.slots[t0 + i] = slot[i];
        }
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
