// Attention of drafted nodes over a paged bf16 cache, on tcgen05.
//
//   o_i = sum_j softmax_j(q_i . k_j / sqrt(D)) v_j
//
// over the context keys and the nodes whose bit is set in row i's mask, in
// one pass over the keys with a running maximum and sum (log2 units):
//   m' = max(m, max_j s_j),  l' = l 2^(m-m') + sum_j 2^(s_j-m'),
//   o' = o 2^(m-m') + sum_j 2^(s_j-m') v_j.
//
// Work. The rows of one (sequence, KV head) are its nodes times the query
// heads of the group: a Q tile stacks 128 / group nodes, node-major, into the
// 128 rows of an MMA, so K and V are read once for all heads of the group. An
// item is up to two Q tiles (A and B). Where an item has one tile, its two
// softmax groups take alternate key tiles of the same rows and join their
// (o, m, l) at the end; where it has two, they share each key tile. The key
// tiles (128 keys) of all items lie on one axis that is cut into equal shares,
// one per CTA, one CTA per SM: ragged batches and a single long sequence fill
// the GPU alike. An item cut by a share's end leaves partial (o, m, l) in the
// workspace and tree_merge_kernel joins them, always in the same order.
//
// A CTA (three warpgroups):
//   warps 0, 2 TMA producers of Q and K, and of V: boxes [64 dims, group
//              heads, nodes] of Q, boxes of up to 64 keys of one page, through
//              a ring of single K or V tiles in the order the MMAs use them;
//   warp 1     owns TMEM; one lane issues S = Q K^T (128 x 128) and O += P V
//              for jobs i = 0, 1, 2, ... of the groups i % 2, so one group's
//              products run during the other's softmax;
//   warp 3     scheduler: cuts the CTA's share into segments (a run of key
//              tiles of one item) and publishes them ahead in a queue;
//   warps 4-11 two softmax groups, one thread per row: read the S row from
//              TMEM 64 keys at a time, mask, exponentials, P as bf16 into
//              TMEM (the A operand of PV is read from there). The reference m
//              (P, l and O share it, so the quotient is the same) is set by
//              the largest of a row's first scores and moves, by whole log2
//              units, only when a score lies 2^8 above, so a tile usually
//              takes one pass over S: exponentials about the old m and the
//              maximum beside them. O, l and P are rescaled, by a power of
//              two, only when m moves. m lies a whole number of units above
//              that score, so its P is a power of two, which bf16 holds (a row
//              that sees one key returns its value), and so far above that the
//              P of all keys sum to at most 1, whatever comes before the next
//              move: O stays within the largest |v|, so finite values never
//              overflow it.
// P is rounded to bf16 because the tensor cores multiply bf16; sums,
// statistics and O stay f32. Over many rows P's roundings add as much error as
// the output's. A call of few rows, where one row with an unlucky rounding of
// its largest weight shows, has time for a second product per tile (REST): what
// bf16 leaves off, as bf16 again, is multiplied too (P to 2^-15 instead of
// 2^-8), and the output is as exact as its own rounding.
// With head_dim 64 TMEM has columns of its own for P, so without REST S(i + 2)
// is computed while the softmax of S(i) still runs; otherwise P, or what it
// leaves off, takes S's columns and S(i + 2) follows PV(i).
//
// Cells that a row must not see never reach it: their scores are replaced
// before the softmax, and a tile that holds any (nodes, the end of the
// sequence, a window, a page outside the pool) has the V rows that hold no
// position zeroed in shared memory, where P = 0 times a stale NaN would not
// stay 0. A node's own non-finite V is zeroed there as well, and added to the
// rows that do see it after the products (patch_row).
//
// Bounds and times (B200, the join included). One sequence, 708 keys, 14/2
// heads of 64: 12.5 .. 13 us, latency (attention 8, the join's launch 1, the join
// 4). One sequence, 64 nodes at 32.7k keys: 28 us (267 TFLOP/s). 32 sequences of
// 128 .. 8k keys with up to 16 nodes, 28/4 heads of 128: 66 us, 4.5 TB/s, bound
// by the loads. 64 sequences of 3k .. 8k keys with 40 .. 64 nodes: 433 .. 445 us,
// 625 TFLOP/s; there the chain S, softmax, PV of a tile (about 4400 cycles for the
// two groups, of which the products are 2100 and the exponentials 2000) and
// the clock under the power limit (1.62 of 1.96 GHz) bound it. S two jobs
// ahead in 64-key tiles, with one MMA warp or one per group, was slower (470
// .. 480 us: twice the waits, each 60 .. 200 cycles beside two busy warps per
// scheduler), as was handing S and P over in halves (486 us).
//
// All mbarrier waits are bounded: on a timeout the CTA waits (bounded) for its
// own copies and MMAs in flight, frees its TMEM and exits, and the join makes
// every row NaN.
#pragma once

#include "attention_mma.cuh"
#include "common.cuh"
#include "pair.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace cheetah {

constexpr int kTreeKeys = 128;      // keys per tile
constexpr int kTreeRows = 128;      // rows of a Q tile
constexpr int kTreeThreads = 384;   // warpgroups: loads and MMAs, softmax A, softmax B
constexpr int kTreeHeadroomLog2 = 8;
constexpr int kTreeMergeThreads = 256;
constexpr int kTreeMergeCtas = 4;     // per SM
constexpr int kTreeMergeWarps = kTreeMergeThreads / kWarp;
constexpr int kTreeMaxCtas = 256;     // CTAs of the attention launch that a merge can list
// Registers per thread after the split of the launch's 168: 128 x 64 + 256 x
// 216 is below 384 x 168.
constexpr int kTreeLeanRegs = 64, kTreeSoftmaxRegs = 216;
static_assert(128 * kTreeLeanRegs + 256 * kTreeSoftmaxRegs <= kTreeThreads * 168, "register split");

template <int HD>
struct TreeCfg {
    static constexpr int kHalves = HD / 64;
    static constexpr int kHalfBytes = kTreeKeys * 128;   // 64 dimensions of a tile
    static constexpr int kTile = kTreeKeys * HD * 2;     // one K, V or Q tile
    static constexpr int kBufs = HD == 64 ? 12 : 5;      // ring
    static constexpr int kTiles = 2 * kTile + kBufs * kTile;
    // Cost units of the shares: a key tile of an item with one Q tile (bound
    // by its loads) and with two (by the products and exponentials), and an
    // item's beginning and end. Halves of a
    // one-tile key tile's time, fitted to measured times.
    static constexpr int kOne = 2, kTwo = HD == 64 ? 4 : 3, kItem = HD == 64 ? 8 : 6;
    static constexpr int kMinShare = 4;
    static_assert(kMinShare >= kTwo, "every share holds a tile");
    // TMEM columns: S_A | S_B | O_A | O_B and, where they fit, P_A | P_B;
    // else P takes the columns of the S it came from.
    static constexpr bool kOwnP = HD == 64;
    static constexpr uint32_t kOCol = 2 * kTreeKeys;
    static constexpr uint32_t kPCol = kOwnP ? kOCol + 2 * HD : 0;
    static constexpr uint32_t kPStep = kOwnP ? kTreeKeys / 2 : kTreeKeys;  // columns from P_A to P_B
    static constexpr uint32_t kPHalf = kOwnP ? 32 : 64;                    // from the first 64 keys' to the rest's
    // What bf16 leaves off of P, 32 columns of each half of S.
    static constexpr uint32_t kRestCol = 32;
    static_assert((kOwnP ? kPCol + kTreeKeys : kOCol + 2 * HD) <= 512, "TMEM columns");
};

// What a split item needs to be joined, written by the CTA that begins it.
struct TreeSplit {
    int row0, nodes, kvh;
    int first_slot;  // of the beginning; the other parts are slot 0 of the next CTAs
    int parts;       // 0: nothing to join; -1: the CTA gave up
    int pad[3];
};

struct TreeAttnParams {
    const int32_t *page_table;
    int max_pages, num_pages, page_tokens, box_keys;
    const int32_t *seq_lens, *row_starts;
    int batch, rows;
    const uint32_t *tree_mask;  // [rows][mask_words32]
    int mask_words32;
    const int32_t *positions;
    int window;
    int q_heads, kv_heads, group, tile_nodes;
    float scale_log2;
    const uint16_t *v_pool;
    uint16_t *out;
    TreeSplit *splits;  // [CTAs]
    float4 *part_o;     // [CTAs][2][HD/4][256] unnormalised: lanes (rows) write and read side by side
    float2 *part_ml;    // [CTAs][2][256]
};

// A run of key tiles [t0, t1) of one item.
struct TreeSegment {
    int row0, n;           // the sequence's first row and row count
    int ctx, len;          // context keys; cached positions within the table
    int b, kvh;
    int node0, nodes;      // the item's nodes within the sequence
    int t0, t1;
    int jobs;              // MMA jobs (0: rows to be zeroed; -1: no more segments)
    int two_tiles;
    int low;               // first key any row may see
    int slot;              // workspace slot of a part; -1: the segment is its whole item
};

// Rows, context and tile range of sequence b.
struct TreeSeq {
    int row0, n, ctx, len, low, tile_lo, tiles;
    int pairs;  // items of two Q tiles
    int items;  // pairs, and one of a single Q tile where nodes are left for it
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeAttnParams &p, int b) {
    TreeSeq s;
    const int r0 = p.row_starts[b], r1 = p.row_starts[b + 1], len = p.seq_lens[b];
    s.row0 = min(max(r0, 0), p.rows);
    s.n = max(min(r1, p.rows) - s.row0, 0);
    s.ctx = len - s.n;
    s.len = (int)min((long long)len, (long long)p.max_pages * p.page_tokens);
    s.low = p.window > 0 ? max(0, s.ctx - p.window + 1) : 0;
    s.tile_lo = s.low / kTreeKeys;
    // Without room for its rows a sequence's items are one tile that writes zeros.
    s.tiles = s.ctx < 0 ? 1 : max(1, (s.len + kTreeKeys - 1) / kTreeKeys - s.tile_lo);
    const int rest = s.n % (2 * p.tile_nodes);
    s.pairs = s.n / (2 * p.tile_nodes) + (rest > p.tile_nodes);
    s.items = s.pairs + (rest > 0 && rest <= p.tile_nodes);
    return s;
}
template <int HD>
__device__ __forceinline__ int tree_item_units(const TreeSeq &s, bool two) {
    return TreeCfg<HD>::kItem + s.tiles * (two ? TreeCfg<HD>::kTwo : TreeCfg<HD>::kOne);
}
// Units of one KV head of a sequence.
template <int HD>
__device__ __forceinline__ int tree_head_units(const TreeSeq &s) {
    return s.pairs * tree_item_units<HD>(s, true) + (s.items - s.pairs) * tree_item_units<HD>(s, false);
}
template <int HD>
__device__ __forceinline__ int tree_units(const TreeAttnParams &p, int b) {
    return tree_head_units<HD>(tree_seq(p, b)) * p.kv_heads;
}

// The ring position of tile i's K and V within a segment of T tiles, in the
// order of first use. Both groups on each tile: K0 V0 K1 V1 .., or K0 K1 V0
// K2 V1 .. with S a job ahead; alternating groups: K0 K1 V0 K2 V1 K3 .., or
// K0 K1 K2 V0 K3 V1 ...
template <bool kAhead>
__device__ __forceinline__ int tree_pos_k(bool two, int i) {
    if (kAhead) return two ? max(2 * i - 1, 0) : (i < 2 ? i : 2 * i - 2);
    return two ? 2 * i : (i < 2 ? i : 2 * i - 1);
}
template <bool kAhead>
__device__ __forceinline__ int tree_pos_v(bool two, int i, int T) {
    if (kAhead) return two ? min(2 * i + 2, 2 * T - 1) : min(2 * i + 3, T + i);
    return two ? 2 * i + 1 : min(2 * i + 2, T + i);
}

constexpr int kTreeQueue = 4;              // segments the scheduler may be ahead
constexpr int kTreeQueueReaders = 3 + 8;   // two producers, the MMA thread, the softmax warps
struct TreeShared {
    uint64_t full[12], empty[12];
    uint64_t seg_full[kTreeQueue], seg_empty[kTreeQueue];
    uint64_t q_full, q_empty, s_full[2], s_free[2], p_full[2], pv_done[2], seg_done, exchange, drain;
    TreeSegment queue[kTreeQueue];
    uint32_t tmem;
    int abort_flag, non_finite;
    uint32_t valid[12];  // per ring buffer: which 16-key parts of V hold loaded positions
    float2 ml[2][kTreeRows];
};

template <int HD>
constexpr size_t tree_attention_smem() { return (size_t)TreeCfg<HD>::kTiles + 3 * 1024; }
static_assert(sizeof(TreeShared) <= 3 * 1024, "fits behind the tiles");

// The role's next segment, once the scheduler has published it; false at the
// end of the share or when a wait gave up (then *ok is false).
__device__ __forceinline__ bool tree_next(TreeShared &sh, int seg, bool &ok) {
    ok = __all_sync(__activemask(), mbar_wait(smem_u32(&sh.seg_full[seg % kTreeQueue]), (seg / kTreeQueue) & 1));
    return ok && sh.queue[seg % kTreeQueue].jobs >= 0;
}
__device__ __forceinline__ void tree_release(TreeShared &sh, int seg) { mbar_arrive(smem_u32(&sh.seg_empty[seg % kTreeQueue])); }

// Bits js .. js+31 of a row's mask (js may be negative or past the end).
__device__ __forceinline__ uint32_t tree_mask_bits(const uint32_t *mask, int words, int js) {
    const int w = js >> 5, o = js & 31;
    const uint32_t lo = w >= 0 && w < words ? mask[w] : 0u;
    const uint32_t hi = w + 1 >= 0 && w + 1 < words ? mask[w + 1] : 0u;
    return __funnelshift_r(lo, hi, o);
}
// The low `n` bits (n clamped to 0..32).
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : (n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u); }

// Keys p0 .. p0+31 that row `row` sees (pages aside).
__device__ __forceinline__ uint32_t tree_visible(const TreeAttnParams &p, const TreeSegment &g, int row, int p0) {
    uint32_t bits = low_bits(g.ctx - p0);
    int low = 0;
    if (p.window > 0) {
        low = max(p.positions[row], g.ctx) - p.window + 1;
        bits &= ~low_bits(low - p0);
    }
    if (p0 + 32 > g.ctx) {
        uint32_t nodes = tree_mask_bits(p.tree_mask + (long long)row * p.mask_words32, p.mask_words32, p0 - g.ctx) &
                         ~low_bits(g.ctx - p0) & low_bits(g.ctx + g.n - p0);
        if (p.window > 0) {
            for (uint32_t rest = nodes; rest;) {
                const int i = __ffs(rest) - 1;
                rest &= rest - 1;
                if (max(p.positions[g.row0 + p0 + i - g.ctx], g.ctx) < low) nodes &= ~(1u << i);
            }
        }
        bits |= nodes;
    }
    return bits & low_bits(g.len - p0);
}

__device__ __forceinline__ bool bf16_non_finite(uint32_t half) { return (half & 0x7F80u) == 0x7F80u; }

// acc + 0 * w: stays zero while the values are finite.
__device__ __forceinline__ uint32_t probe_bf16x2(uint32_t w, uint32_t acc) {
    uint32_t r;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(w), "r"(0u), "r"(acc));
    return r;
}

// One V row of a masked tile in shared memory, of a key that some row does not
// see: zero where it holds no position, finite elsewhere (its non-finite
// values are noted for patch_row).
template <int HD>
__device__ __forceinline__ void tree_clean_v(TreeShared &sh, uint8_t *v_row, bool holds) {
    // Each lane begins at another cell: the rows lie 128 bytes apart.
    auto cell = [&](int c) -> uint4 & {
        return *reinterpret_cast<uint4 *>(v_row + (c >> 3) * TreeCfg<HD>::kHalfBytes + ((c + threadIdx.x) & 7) * 16);
    };
    if (!holds) {
#pragma unroll
        for (int c = 0; c < HD / 8; ++c) cell(c) = make_uint4(0u, 0u, 0u, 0u);
    } else {
        uint32_t acc[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int c = 0; c < HD / 8; ++c) {
            const uint4 v = cell(c);
            acc[0] = probe_bf16x2(v.x, acc[0]);
            acc[1] = probe_bf16x2(v.y, acc[1]);
            acc[2] = probe_bf16x2(v.z, acc[2]);
            acc[3] = probe_bf16x2(v.w, acc[3]);
        }
        if (!((acc[0] | acc[1] | acc[2] | acc[3]) & 0x7FFF7FFFu)) return;
        *reinterpret_cast<volatile int *>(&sh.non_finite) = 1;
        __threadfence_block();  // flag before the zeros that hide it from the other group
#pragma unroll 1
        for (int c = 0; c < HD / 8; ++c) {
            const uint4 v = cell(c);
            uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                if (bf16_non_finite(w[x])) w[x] &= 0xFFFF0000u;
                if (bf16_non_finite(w[x] >> 16)) w[x] &= 0x0000FFFFu;
            }
            cell(c) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Adds the non-finite values of the V rows that `row` sees in [t0, t1) to the
// result this thread's warp has just stored (columns d0 .. d0+cols). Their
// products were left out of the MMAs.
template <int HD>
__device__ __noinline__ void patch_row(const TreeAttnParams &p, const TreeSegment &g, int row, int d0, int cols,
                                       uint16_t *out, float *part) {
    // Without a window the context was left alone (adding its values again, in
    // the tile of the first node, changes nothing).
    const int begin = p.window > 0 ? g.t0 * kTreeKeys : max(g.t0 * kTreeKeys, g.ctx / kTreeKeys * kTreeKeys);
    for (int p0 = begin; p0 < min(g.t1 * kTreeKeys, g.len); p0 += 32) {
        for (uint32_t rest = tree_visible(p, g, row, p0); rest; rest &= rest - 1) {
            const int pos = p0 + __ffs(rest) - 1;
            const int page = p.page_table[(long long)g.b * p.max_pages + pos / p.page_tokens];
            if (page < 0 || page >= p.num_pages) continue;
            const uint16_t *v = p.v_pool + (((long long)page * p.kv_heads + g.kvh) * p.page_tokens + pos % p.page_tokens) * HD;
            for (int d = d0; d < d0 + cols; ++d) {
                if (!bf16_non_finite(v[d])) continue;
                if (part) part[(d / 4) * 1024 + d % 4] += bf16_to_f32(v[d]);
                else out[d] = f32_to_bf16_rne(bf16_to_f32(out[d]) + bf16_to_f32(v[d]));
            }
        }
    }
}

// Products of two bf16 pairs (exact for powers of two within range).
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Exponentials of 64 scores about m as bf16 pairs, their sum (as two) and the
// largest score. REST: the pairs, and what bf16 leaves off of them, go to TMEM
// 16 at a time instead of to w (which would not fit the registers).
template <bool REST>
__device__ __forceinline__ float tree_exponentials(const float (&sc)[64], unsigned long long scale2, float neg_m, uint32_t (&w)[32],
                                                   float &s0, float &s1, uint32_t p_addr, uint32_t rest_addr) {
    const unsigned long long neg_m2 = pair_f32(neg_m, neg_m);
    unsigned long long sums[4] = {0ull, 0ull, 0ull, 0ull};
    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        uint32_t cut[16], rest[16];
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            const int k = 16 * c + x;
            mx[k & 3] = max3(mx[k & 3], sc[2 * k], sc[2 * k + 1]);
            float e0, e1;
            unpair_f32(fma_pair(pair_f32(sc[2 * k], sc[2 * k + 1]), scale2, neg_m2), e0, e1);
            e0 = fast_exp2(e0);
            e1 = fast_exp2(e1);
            sums[k & 3] = add_pair(sums[k & 3], pair_f32(e0, e1));
            if constexpr (REST) {
                // Cut off, not rounded, and the rest made larger by e 2^-23: it
                // is positive like e, so an infinite V gives no inf - inf or 0 inf.
                const uint32_t b0 = __float_as_uint(e0) & 0xFFFF0000u, b1 = __float_as_uint(e1) & 0xFFFF0000u;
                cut[x] = b0 >> 16 | b1;
                rest[x] = pack_bf16(fmaf(e0, 1.0f + 0x1p-23f, -__uint_as_float(b0)), fmaf(e1, 1.0f + 0x1p-23f, -__uint_as_float(b1)));
            } else {
                w[k] = pack_bf16(e0, e1);
            }
        }
        if constexpr (REST) {
            tmem_st16_nowait(p_addr + c * 16, cut);
            tmem_st16_nowait(rest_addr + c * 16, rest);
        }
    }
    unpair_f32(add_pair(add_pair(sums[0], sums[1]), add_pair(sums[2], sums[3])), s0, s1);
    return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
}

// Stores 64 bytes of each lane's row (four 16-byte cells), with the four cells
// of a row written by neighbouring lanes: lane l's v[j] becomes lane j's v[l]
// among each four lanes, so a store covers 8 rows instead of 32.
__device__ __forceinline__ void store_rows4(uint16_t *dst, uint32_t (&v)[4][4], uint32_t live_mask) {
    const int lane = threadIdx.x % kWarp;
#pragma unroll
    for (int s = 1; s < 4; s <<= 1) {
        const bool high = lane & s;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j & s) continue;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const uint32_t got = __shfl_xor_sync(0xFFFFFFFFu, high ? v[j][x] : v[j | s][x], s);
                if (high) v[j][x] = got;
                else v[j | s][x] = got;
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int from = (lane & ~3) + j;
        uint16_t *row = reinterpret_cast<uint16_t *>(__shfl_sync(0xFFFFFFFFu, reinterpret_cast<unsigned long long>(dst), from));
        if (live_mask >> from & 1)
            *reinterpret_cast<uint4 *>(row + (lane & 3) * 8) = make_uint4(v[j][0], v[j][1], v[j][2], v[j][3]);
    }
}

template <int HD, bool REST>
__global__ void __launch_bounds__(kTreeThreads, 1)
    tree_attention_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                          const __grid_constant__ CUtensorMap v_map, const TreeAttnParams p) {
    using C = TreeCfg<HD>;
    constexpr bool kAhead = C::kOwnP && !REST;  // S(i + 2) before PV(i)
    constexpr uint32_t kIdescS = umma_idesc_bf16(kTreeRows, kTreeKeys);
    constexpr uint32_t kIdescPV = umma_idesc_bf16(kTreeRows, HD) | (1u << 16);  // V MN-major
    // The kernel's only shared memory, so it begins at a 1024-byte boundary
    // (the swizzled tiles' alignment).
    extern __shared__ __align__(1024) uint8_t tree_smem[];
    uint8_t *q_s = tree_smem, *ring = tree_smem + 2 * C::kTile;
    TreeShared &sh = *reinterpret_cast<TreeShared *>(tree_smem + C::kTiles);
    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::kBufs; ++i) {
            mbar_init(smem_u32(&sh.full[i]), 1);
            mbar_init(smem_u32(&sh.empty[i]), 1);
        }
        for (int i = 0; i < kTreeQueue; ++i) {
            mbar_init(smem_u32(&sh.seg_full[i]), 1);
            mbar_init(smem_u32(&sh.seg_empty[i]), kTreeQueueReaders);
        }
        mbar_init(smem_u32(&sh.q_full), 1);
        mbar_init(smem_u32(&sh.q_empty), 1);
        for (int g = 0; g < 2; ++g) {
            mbar_init(smem_u32(&sh.s_full[g]), 1);
            mbar_init(smem_u32(&sh.s_free[g]), 4);
            mbar_init(smem_u32(&sh.p_full[g]), 4);
            mbar_init(smem_u32(&sh.pv_done[g]), 1);
        }
        mbar_init(smem_u32(&sh.seg_done), 1);
        mbar_init(smem_u32(&sh.exchange), 8);
        mbar_init(smem_u32(&sh.drain), 1);
        sh.abort_flag = 0;
        sh.non_finite = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                     "r"(512u));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    pdl_wait();

    int ring_at = 0;   // ring positions of the segments before
    int issued = 0;    // producers: tiles requested are at positions below this
    int q_issued = 0;
    if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTreeLeanRegs));
    if (warp == 3) {
        // Scheduler. Total units, and the sequence in which this CTA's share
        // begins (the host has checked that the units of any lengths fit 31
        // bits); a lane per sequence, other warps wait for the first segment.
        int total = 0, mine = 0;
        for (int b = lane; b < p.batch; b += kWarp) {
            const int units = tree_units<HD>(p, b);
            if (b == lane) mine = units;
            total += units;
        }
        total = __reduce_add_sync(0xFFFFFFFFu, total);
        const int share = max(C::kMinShare, (int)(((unsigned)total + gridDim.x - 1) / gridDim.x));
        const int u0 = (int)min((long long)blockIdx.x * share, (long long)total);
        int start = -1, before = 0;
        int at = 0;  // unit within the sequence, then within the item
        for (int b0 = 0; b0 < p.batch && start < 0 && u0 < total; b0 += kWarp) {
            const int b = b0 + lane;
            const int units = b0 == 0 ? mine : (b < p.batch ? tree_units<HD>(p, b) : 0);
            int end = units;
#pragma unroll
            for (int o = 1; o < kWarp; o <<= 1) {
                const int up = __shfl_up_sync(0xFFFFFFFFu, end, o);
                if (lane >= o) end += up;
            }
            end += before;
            const uint32_t here = __ballot_sync(0xFFFFFFFFu, end - units <= u0 && u0 < end);
            if (here) {
                start = b0 + __ffs(here) - 1;
                at = u0 - __shfl_sync(0xFFFFFFFFu, end - units, __ffs(here) - 1);
            }
            before = __shfl_sync(0xFFFFFFFFu, end, kWarp - 1);
        }
        // It walks over the share's items and publishes its segments.
        if (lane == 0) {
            int b = start, left = min(share, total - u0), unit = u0, seg = 0;
            TreeSeq s = {};
            int kvh = 0, rt = 0;
            if (left > 0) {
                s = tree_seq(p, b);
                const int head = tree_head_units<HD>(s), pair = tree_item_units<HD>(s, true);
                kvh = at / head;
                at -= kvh * head;
                rt = min(at / pair, s.pairs);
                at -= rt * pair;
            }
            TreeSplit split = {};
            bool ok = true;
            while (true) {
                TreeSegment g = {};
                g.jobs = -1;
                while (left > 0) {
                    const bool two = rt < s.pairs;
                    const int units = tree_item_units<HD>(s, two), cost = two ? C::kTwo : C::kOne;
                    const int take = min(left, units - at);
                    // Tiles of this piece; an item's first kItem units hold none.
                    const int t0 = max(at - C::kItem, 0) / cost, t1 = max(at + take - C::kItem, 0) / cost;
                    if (t1 > t0) {
                        const bool whole = t1 - t0 == s.tiles;
                        g.row0 = s.row0;
                        g.n = s.n;
                        g.ctx = s.ctx;
                        g.len = s.len;
                        g.b = b;
                        g.kvh = kvh;
                        g.node0 = rt * 2 * p.tile_nodes;
                        g.nodes = min(s.n - g.node0, 2 * p.tile_nodes);
                        g.two_tiles = two;
                        g.t0 = s.tile_lo + t0;
                        g.t1 = s.tile_lo + t1;
                        g.jobs = s.ctx < 0 ? 0 : (two ? 2 : 1) * (t1 - t0);
                        g.low = s.low;
                        g.slot = whole ? -1 : (seg == 0 ? 0 : 1);
                        if (t0 == 0 && !whole) {
                            split.row0 = s.row0 + g.node0;
                            split.nodes = g.nodes;
                            split.kvh = kvh;
                            split.first_slot = g.slot;
                            // Within the grid even if sequences share rows, which the units do not count on.
                            split.parts = min((unit - at + units - 1) / share - (int)blockIdx.x + 1, (int)(gridDim.x - blockIdx.x));
                        }
                    }
                    unit += take;
                    left -= take;
                    at += take;
                    if (at == units) {
                        at = 0;
                        if (++rt == s.items) {
                            rt = 0;
                            ++kvh;
                        }
                        while (left > 0 && kvh >= (s.items > 0 ? p.kv_heads : 0)) {  // the next sequence with rows
                            if (++b >= p.batch) {
                                left = 0;
                                break;
                            }
                            s = tree_seq(p, b);
                            kvh = 0;
                        }
                    }
                    if (t1 > t0) break;
                }
                ok = mbar_wait(smem_u32(&sh.seg_empty[seg % kTreeQueue]), ((seg / kTreeQueue) & 1) ^ 1);
                if (!ok) break;
                sh.queue[seg % kTreeQueue] = g;
                mbar_arrive(smem_u32(&sh.seg_full[seg % kTreeQueue]));
                ++seg;
                if (g.jobs < 0) break;
            }
            p.splits[blockIdx.x] = split;
            if (!ok) sh.abort_flag = 1;
        }
    } else if (warp == 0 || warp == 2) {
        // Producers: warp 0 loads Q and K tiles, warp 2 V tiles.
        const bool is_v = warp == 2;
        const CUtensorMap *map = is_v ? &v_map : &k_map;
        const int boxes = kTreeKeys / p.box_keys;
        bool ok = true;
        // Q, once the previous segment's S products are done (in the first
        // segment before the keys, later behind the first of them).
        auto load_q = [&](const TreeSegment &g) -> bool {
            if (!__all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&sh.q_empty), (q_issued & 1) ^ 1))) return false;
            if (lane == 0) {
                const int tiles = g.two_tiles ? 2 : 1;
                mbar_expect_tx(smem_u32(&sh.q_full), (uint32_t)(tiles * C::kHalves * p.group * p.tile_nodes * 128));
                for (int t = 0; t < tiles; ++t) {
                    for (int h = 0; h < C::kHalves; ++h) {
                        tma_load_3d(smem_u32(q_s + t * C::kTile + h * C::kHalfBytes), &q_map, h * 64, g.kvh * p.group,
                                    g.row0 + g.node0 + t * p.tile_nodes, smem_u32(&sh.q_full));
                    }
                }
            }
            ++q_issued;
            return true;
        };
        for (int seg = 0; tree_next(sh, seg, ok); ++seg) {
            const TreeSegment &g = sh.queue[seg % kTreeQueue];
            const int T = g.t1 - g.t0;
            const bool two = g.two_tiles;
            const int len = g.len, low = g.low, kvh = g.kvh, t0 = g.t0;
            const int32_t *table = p.page_table + (long long)g.b * p.max_pages;
            if (g.jobs > 0) {
                // Pool rows of 32 consecutive boxes, one per lane (-1: not
                // loaded); a tile's boxes never straddle them (32 is a
                // multiple of 2, 4 and 8).
                int first = -kWarp, my_row = -1;
                uint32_t loaded = 0;
                if (!is_v && seg == 0) load_q(g);
                for (int i = 0; i < T; ++i) {
                    const int at = ring_at + (is_v ? tree_pos_v<kAhead>(two, i, T) : tree_pos_k<kAhead>(two, i));
                    const int buf = at % C::kBufs;
                    const int box0 = (t0 + i) * boxes;
                    if (box0 >= first + kWarp) {
                        first = box0;
                        const long long pos = (long long)(box0 + lane) * p.box_keys;
                        my_row = -1;
                        if (pos < len && pos + p.box_keys > low) {
                            const int col = (int)pos / p.page_tokens;
                            const int page = table[col];
                            if (page >= 0 && page < p.num_pages)
                                my_row = (page * p.kv_heads + kvh) * p.page_tokens + ((int)pos - col * p.page_tokens);
                        }
                        loaded = __ballot_sync(0xFFFFFFFFu, my_row >= 0);
                    }
                    ok = __all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&sh.empty[buf]), ((at / C::kBufs) & 1) ^ 1));
                    if (!ok) break;
                    const uint32_t good = (loaded >> (box0 - first)) & low_bits(boxes);
                    const uint32_t bar = smem_u32(&sh.full[buf]);
                    const uint32_t dst = smem_u32(ring + buf * C::kTile);
                    if (lane == 0) {
                        if (is_v) {
                            uint32_t valid = 0;
                            for (int x = 0; x < boxes; ++x) {
                                if (good >> x & 1) valid |= low_bits(8 / boxes) << (x * (8 / boxes));
                            }
                            sh.valid[buf] = valid;
                        }
                        mbar_expect_tx(bar, (uint32_t)(__popc(good) * p.box_keys * HD * 2));
                    }
                    for (int x = 0; x < boxes; ++x) {
                        const int row = __shfl_sync(0xFFFFFFFFu, my_row, box0 - first + x);
                        if (lane == 0 && row >= 0) {
#pragma unroll
                            for (int h = 0; h < C::kHalves; ++h)
                                tma_load_2d(dst + h * C::kHalfBytes + x * p.box_keys * 128, map, h * 64, row, bar);
                        }
                    }
                    issued = at + 1;
                    if (!is_v && seg > 0 && i == min(1, T - 1) && !load_q(g)) {
                        ok = false;
                        break;
                    }
                }
                ring_at += 2 * T;
            }
            if (!ok) break;
            __syncwarp();
            if (lane == 0) tree_release(sh, seg);
        }
        if (!ok) sh.abort_flag = 1;
    } else if (warp == 1) {
        // The whole warp walks, one elected lane issues.
        const bool leader = elect_one();
        uint32_t q_phase = 0, p_phase[2] = {0, 0}, free_phase[2] = {0, 0};
        // The next ring position; buffers are first used in ring order.
        int next_buf = 0;
        uint32_t next_phase = 0;
        int k_buf = 0, v_buf = 0;
        const uint64_t q_desc = umma_smem_desc(smem_u32(q_s));
        const uint64_t k_desc = umma_smem_desc(smem_u32(ring));
        const uint64_t v_desc = umma_smem_desc_mn(smem_u32(ring), HD > 64 ? C::kHalfBytes : 16);
        bool ok = true;
        auto wait = [&](uint64_t &bar, uint32_t phase) -> bool { return __all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&bar), phase)); };
        auto take = [&](int &buf) -> bool {
            buf = next_buf;
            const bool landed = wait(sh.full[buf], next_phase);
            if (++next_buf == C::kBufs) {
                next_buf = 0;
                next_phase ^= 1;
            }
            return landed;
        };
        for (int seg = 0; tree_next(sh, seg, ok); ++seg) {
            const bool two = sh.queue[seg % kTreeQueue].two_tiles;
            const int jobs = sh.queue[seg % kTreeQueue].jobs;
            auto issue_s = [&](int i) -> bool {
                const int grp = i & 1;
                if ((!two || grp == 0) && !take(k_buf)) return false;
                tc_fence_after();
                const uint64_t qd = q_desc + (two ? grp * (C::kTile >> 4) : 0);
                const uint64_t kd = k_desc + (uint32_t)(k_buf * (C::kTile >> 4));
                if (leader) {
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k) {
                        const uint32_t off = (uint32_t)((k >> 2) * C::kHalfBytes + (k & 3) * 32) >> 4;
                        umma_bf16(tmem + grp * kTreeKeys, qd + off, kd + off, kIdescS, k > 0 ? 1u : 0u);
                    }
                    umma_commit(smem_u32(&sh.s_full[grp]));
                    if (!two || grp == 1) umma_commit(smem_u32(&sh.empty[k_buf]));
                    if (i == jobs - 1) umma_commit(smem_u32(&sh.q_empty));
                }
                __syncwarp();
                return true;
            };
            auto issue_pv = [&](int i) -> bool {
                const int grp = i & 1;
                if ((!two || grp == 0) && !take(v_buf)) return false;
                const uint64_t vd = v_desc + (uint32_t)(v_buf * (C::kTile >> 4));
                if (!wait(sh.p_full[grp], p_phase[grp])) return false;
                p_phase[grp] ^= 1;
                tc_fence_after();
                if (leader) {
#pragma unroll
                    for (int k = 0; k < kTreeKeys / 16; ++k) {
                        umma_bf16_ta(tmem + C::kOCol + grp * HD, tmem + C::kPCol + grp * C::kPStep + (k >> 2) * C::kPHalf + (k & 3) * 8,
                                     vd + (k * 2048 >> 4), kIdescPV, (i > 1 || k > 0) ? 1u : 0u);
                    }
                    if constexpr (REST) {
#pragma unroll
                        for (int k = 0; k < kTreeKeys / 16; ++k) {
                            umma_bf16_ta(tmem + C::kOCol + grp * HD, tmem + grp * kTreeKeys + (k >> 2) * 64 + C::kRestCol + (k & 3) * 8,
                                         vd + (k * 2048 >> 4), kIdescPV, 1u);
                        }
                    }
                    if (C::kOwnP) umma_commit(smem_u32(&sh.pv_done[grp]));
                    if (!two || grp == 1) umma_commit(smem_u32(&sh.empty[v_buf]));
                    if (i == jobs - 1) umma_commit(smem_u32(&sh.seg_done));
                }
                __syncwarp();
                return true;
            };
            // S(i + 2) goes into S(i)'s columns: once the softmax has read
            // them, or, where P or what it leaves off lies there, behind PV(i).
            auto free_s = [&](int i) -> bool { return wait(sh.s_free[i & 1], free_phase[i & 1]); };
            if (jobs > 0) {
                ok = wait(sh.q_full, q_phase);
                q_phase ^= 1;
                if (ok) ok = issue_s(0) && (jobs < 2 || issue_s(1));
                for (int i = 0; ok && i < jobs; ++i) {
                    if (kAhead) {
                        if (i + 2 < jobs) ok = free_s(i) && issue_s(i + 2);
                        free_phase[i & 1] ^= 1;
                        ok = ok && issue_pv(i);
                    } else {
                        ok = issue_pv(i) && (i + 2 >= jobs || issue_s(i + 2));
                    }
                }
                if (!ok) break;
            }
            if (lane == 0) tree_release(sh, seg);
            __syncwarp();
        }
        if (!ok) sh.abort_flag = 1;
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTreeSoftmaxRegs));
        const int grp = (warp - 4) / 4, quad = warp % 4;
        const int r = quad * 32 + lane;
        const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
        const uint32_t s_addr = tmem + lane_off + grp * kTreeKeys;
        const uint32_t o_addr = tmem + lane_off + C::kOCol + grp * HD;
        const uint32_t p_addr = tmem + lane_off + C::kPCol + grp * C::kPStep;
        const int node_of_r = r / p.group, head_of_r = r % p.group;
        uint32_t s_phase = 0, pv_phase = 0, done_phase = 0, x_phase = 0;
        bool ok = true;
        for (int seg = 0; tree_next(sh, seg, ok); ++seg) {
            const TreeSegment &g = sh.queue[seg % kTreeQueue];
            const int jobs = g.jobs, T = g.t1 - g.t0;
            const bool two = g.two_tiles;
            const int node = g.node0 + (two ? grp * p.tile_nodes : 0) + node_of_r;
            const bool live = node_of_r < p.tile_nodes && node < g.node0 + g.nodes;
            const int row = g.row0 + node;
            uint16_t *out_row = p.out + ((long long)row * p.q_heads + g.kvh * p.group + head_of_r) * HD;
            if (jobs == 0) {
                if (live && (two || grp == 0)) {
#pragma unroll
                    for (int i = 0; i < HD / 8; ++i) reinterpret_cast<uint4 *>(out_row)[i] = make_uint4(0u, 0u, 0u, 0u);
                }
                __syncwarp();
                if (lane == 0) tree_release(sh, seg);
                continue;
            }
            const bool warp_live = __any_sync(0xFFFFFFFFu, live);
            const int ctx = g.ctx;
            // From a score to the m that it sets: log2 of the number of keys,
            // rounded up, and the headroom.
            const float spread = (float)(32 - __clz(g.len - 1));
            float m_run = -INFINITY, l_run = 0.0f;
            for (int i = grp; i < jobs; i += 2) {
                const int tile = two ? i >> 1 : i;
                const int p0 = (g.t0 + tile) * kTreeKeys;
                // What the row sees of a tile that holds nodes or a window's
                // edge, while S is on its way.
                const bool partial = p.window > 0 || p0 + kTreeKeys > ctx;
                uint32_t vis[4] = {0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu};
                if (partial) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) vis[c] = live ? tree_visible(p, g, row, p0 + 32 * c) : 0u;
                }
                if (!__all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&sh.s_full[grp]), s_phase))) {
                    ok = false;
                    break;
                }
                s_phase ^= 1;
                tc_fence_after();
                // The first 64 scores are on their way during the other waits,
                // the second 64 during the first's exponentials.
                float sc[2][64];
                if (warp_live) {
                    tmem_ld32_nowait(s_addr, sc[0]);
                    tmem_ld32_nowait(s_addr + 32, sc[0] + 32);
                }
                const int at = ring_at + tree_pos_v<kAhead>(two, tile, T), buf = at % C::kBufs;
                // V of this tile stays until this group's P is consumed, so
                // its phase cannot have moved on.
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&sh.full[buf]), (at / C::kBufs) & 1));
                // P's columns and O are this thread's once PV(i - 2) is done
                // (where P lies in S's columns, S(i) has come after it).
                if (C::kOwnP) {
                    if (ok && i > 1) ok = __all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&sh.pv_done[grp]), pv_phase ^ 1));
                    pv_phase ^= 1;
                }
                tmem_wait_ld();
                if (!ok) break;
                tc_fence_after();
                const uint32_t valid = sh.valid[buf];
                const bool masked = partial || valid != 0xFFu;
                if (masked) {
                    const bool holds = p0 + r < g.len && (valid >> (r >> 4) & 1);
                    // Every row sees a context key, without a window.
                    if (!holds || p.window > 0 || p0 + r >= ctx) tree_clean_v<HD>(sh, ring + buf * C::kTile + r * 128, holds);
                }
                if (warp_live) {
                    const unsigned long long scale2 = pair_f32(p.scale_log2, p.scale_log2);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (h == REST) {  // with REST the registers are needed until then
                            tmem_ld32_nowait(s_addr + 64, sc[1]);
                            tmem_ld32_nowait(s_addr + 96, sc[1] + 32);
                        }
                        if (h == 1) {
                            tmem_wait_ld();
                            if (kAhead) {
                                tc_fence_before();
                                __syncwarp();
                                if (lane == 0) mbar_arrive(smem_u32(&sh.s_free[grp]));
                            }
                        }
                        if (masked) {
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
                                const uint32_t part = (valid >> (4 * h + 2 * c) & 1 ? 0x0000FFFFu : 0u) |
                                                      (valid >> (4 * h + 2 * c + 1) & 1 ? 0xFFFF0000u : 0u);
                                const uint32_t seen = (h == 0 ? vis[c] : vis[2 + c]) & part;
#pragma unroll
                                for (int k = 0; k < 32; ++k) sc[h][32 * c + k] = (seen >> k & 1) ? sc[h][32 * c + k] : -INFINITY;
                            }
                        }
                        // Exponentials about the present m, and the largest
                        // score beside them; only if it lies too far above m,
                        // m moves and they are done again.
                        uint32_t w[32];
                        float s0, s1;
                        if (i == grp && h == 0) {
                            // The first keys set m.
                            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                            for (int k = 0; k < 32; ++k) mx[k & 3] = max3(mx[k & 3], sc[h][2 * k], sc[h][2 * k + 1]);
                            m_run = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2 + (spread + kTreeHeadroomLog2);
                        }
                        while (true) {
                            const float neg_m = m_run == -INFINITY ? 0.0f : -m_run;
                            const uint32_t p_part = p_addr + h * C::kPHalf, rest = s_addr + h * 64 + C::kRestCol;
                            const float top = p.scale_log2 * tree_exponentials<REST>(sc[h], scale2, neg_m, w, s0, s1, p_part, rest);
                            const bool far = top + spread > m_run;
                            if (!__any_sync(0xFFFFFFFFu, far)) break;
                            // By a whole number, so every rescaling is exact,
                            // and to where `far` is false (from -inf, where the
                            // first keys are unseen: to the score itself).
                            float m_new = m_run;
                            if (far) {
                                // (Once more: a register less outside.)
                                const float to = top + (float)(kTreeHeadroomLog2 + 32 - __clz(g.len - 1));
                                m_new = fmaxf(m_run + ceilf(to - m_run), to);
                            }
                            const float f = m_new == m_run ? 1.0f : exp2f(m_run - m_new);
                            m_run = m_new;
                            l_run *= f;
                            if (h == 1) {
                                const uint32_t f2 = pack_bf16(f, f);
                                tmem_wait_st();
#pragma unroll 1
                                for (int c = 0; c < 2; ++c) {
                                    float pv[16];
                                    tmem_ld16(p_addr + c * 16, pv);
#pragma unroll
                                    for (int k = 0; k < 16; ++k) pv[k] = __uint_as_float(mul_bf16x2(__float_as_uint(pv[k]), f2));
                                    tmem_st16(p_addr + c * 16, pv);
                                    if (!REST) continue;
                                    tmem_ld16(s_addr + C::kRestCol + c * 16, pv);
#pragma unroll
                                    for (int k = 0; k < 16; ++k) pv[k] = __uint_as_float(mul_bf16x2(__float_as_uint(pv[k]), f2));
                                    tmem_st16(s_addr + C::kRestCol + c * 16, pv);
                                }
                            }
                            if (i > 1) {
#pragma unroll 1
                                for (int c = 0; c < HD / 16; ++c) {
                                    float ov[16];
                                    tmem_ld16(o_addr + c * 16, ov);
#pragma unroll
                                    for (int k = 0; k < 16; ++k) ov[k] *= f;
                                    tmem_st16(o_addr + c * 16, ov);
                                }
                            }
                        }
                        l_run += s0 + s1;
                        // In S's columns, P's 32 are among those read by now.
                        if (!REST) {
                            tmem_st16_nowait(p_addr + h * C::kPHalf, w);
                            tmem_st16_nowait(p_addr + h * C::kPHalf + 16, w + 16);
                        }
                    }
                    tmem_wait_st();
                    tc_fence_before();
                } else if (kAhead && lane == 0) {
                    mbar_arrive(smem_u32(&sh.s_free[grp]));
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.p_full[grp]));
            }
            ring_at += 2 * T;
            if (!ok) break;
            if (!__all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&sh.seg_done), done_phase))) {
                ok = false;
                break;
            }
            done_phase ^= 1;
            tc_fence_after();
            // Weights of this row's accumulators: its own, and the other
            // group's where both hold the same row.
            float w_own = 1.0f, w_other = 0.0f, l = l_run, m = m_run;
            if (!two) {
                sh.ml[grp][r] = make_float2(m_run, l_run);
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.exchange));
                if (!__all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&sh.exchange), x_phase))) {
                    ok = false;
                    break;
                }
                x_phase ^= 1;
                const float2 other = sh.ml[grp ^ 1][r];
                m = fmaxf(m_run, other.x);
                w_own = m_run == -INFINITY ? 0.0f : exp2f(m_run - m);
                w_other = other.x == -INFINITY ? 0.0f : exp2f(other.x - m);
                l = l_run * w_own + other.y * w_other;
            }
            if (warp_live) {
                const bool joined = !two && jobs > 1;
                // Where there was one job, only group A has accumulated.
                const uint32_t own = two || joined ? o_addr : tmem + lane_off + C::kOCol;
                const uint32_t other_addr = tmem + lane_off + C::kOCol + (grp ^ 1) * HD;
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                const int slot = g.slot;
                const long long part_row = (long long)(2 * blockIdx.x + max(slot, 0)) * 256 + (two ? grp * kTreeRows : 0) + r;
                float4 *part = p.part_o + (part_row / 256) * (HD / 4) * 256 + part_row % 256;
                const uint32_t live_mask = __ballot_sync(0xFFFFFFFFu, live);
                // Two Q tiles: every column of the own row. One: group A
                // finishes the first half of the columns, B the second.
                const int d0 = two ? 0 : grp * (HD / 2), d1 = two ? HD : d0 + HD / 2;
#pragma unroll 1
                for (int c = d0; c < d1; c += 32) {
                    float ov[32];
                    __syncwarp();  // lanes part at a part's stores; the loads from TMEM are the whole warp's
                    if (joined) {
                        float ox[32];
                        tmem_ld32_nowait(own + c, ov);
                        tmem_ld32_nowait(other_addr + c, ox);
                        tmem_wait_ld();
#pragma unroll
                        for (int k = 0; k < 32; ++k) ov[k] = ov[k] * w_own + ox[k] * w_other;
                    } else {
                        tmem_ld32(own + c, ov);
                    }
                    if (slot >= 0) {
                        if (live) {
#pragma unroll
                            for (int k = 0; k < 8; ++k)
                                part[(c / 4 + k) * 256] = make_float4(ov[4 * k], ov[4 * k + 1], ov[4 * k + 2], ov[4 * k + 3]);
                        }
                    } else {
                        // 64 bytes of a row: 4 lanes write them together.
                        uint32_t v[4][4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
#pragma unroll
                            for (int x = 0; x < 4; ++x) v[k][x] = pack_bf16(ov[8 * k + 2 * x] * inv, ov[8 * k + 2 * x + 1] * inv);
                        }
                        store_rows4(out_row + c, v, live_mask);
                    }
                }
                __syncwarp();  // patch_row reads what the warp has stored
                if (live) {
                    if (slot >= 0 && (two || grp == 0)) p.part_ml[part_row] = make_float2(m, l);
                    if (*reinterpret_cast<volatile int *>(&sh.non_finite))
                        patch_row<HD>(p, g, row, d0, d1 - d0, out_row, slot >= 0 ? reinterpret_cast<float *>(part) : nullptr);
                }
            }
            tc_fence_before();
            // Neither accumulator may be overwritten before both are read, and
            // neither group may fall a segment behind the other's barriers.
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.exchange));
            if (!__all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&sh.exchange), x_phase))) {
                ok = false;
                break;
            }
            x_phase ^= 1;
            if (lane == 0) tree_release(sh, seg);
        }
        if (!ok) sh.abort_flag = 1;
    }
    tc_fence_before();
    __syncthreads();
    // The join may come up from here on; earlier its CTAs would take issue slots
    // from the last softmax rows.
    pdl_launch_dependents();
    if (sh.abort_flag) {
        // A wait gave up: let this CTA's copies and MMAs still in flight land
        // before its shared memory and TMEM are released (bounded waits).
        if ((warp == 0 || warp == 2) && lane == 0) {
            if (q_issued > 0) mbar_wait(smem_u32(&sh.q_full), (q_issued - 1) & 1);
            for (int at = max(0, issued - C::kBufs); at < issued; ++at)
                mbar_wait(smem_u32(&sh.full[at % C::kBufs]), (at / C::kBufs) & 1);
        } else if (warp == 1 && elect_one()) {  // the lane that issued the MMAs
            umma_commit(smem_u32(&sh.drain));
            mbar_wait(smem_u32(&sh.drain), 0);
        }
        if (threadIdx.x == kTreeThreads - 1) p.splits[blockIdx.x].parts = -1;  // the join makes the result NaN
        tc_fence_before();
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
    }
}

// Joins the parts of the items that shares cut: o = sum_k 2^(m_k - m) o_k /
// sum_k 2^(m_k - m) l_k, in a fixed order. The CTAs list the split items and
// share their row blocks. A lane has a row and, where an item has many parts,
// every fourth of them (then a block is 8 rows instead of 32); a warp has
// every eighth column group of four, as the parts lie in the workspace. The
// block is written from shared memory row by row.
template <int HD>
__global__ void __launch_bounds__(kTreeMergeThreads) tree_merge_kernel(const TreeAttnParams p, int ctas) {
    static_assert(kTreeMaxCtas == kTreeMergeThreads, "a thread per listed CTA");
    constexpr int kCols = HD / 4 / kTreeMergeWarps;  // column groups of a warp
    constexpr int kFew = 4;
    __shared__ TreeSplit split_s[kTreeMaxCtas];
    __shared__ int unit_end[kTreeMaxCtas];
    __shared__ int warp_units[kTreeMergeWarps];
    __shared__ uint2 block_s[kWarp][HD / 4 + 1];
    const int tid = threadIdx.x, lane = tid % kWarp, warp = tid / kWarp;
    pdl_wait();
    pdl_launch_dependents();
    int units = 0;
    bool gave_up = false;
    if (tid < ctas) {
        const TreeSplit s = p.splits[tid];
        split_s[tid] = s;
        gave_up = s.parts < 0;
        const int block = s.parts > kFew ? kWarp / 4 : kWarp;
        units = s.parts > 1 ? (s.nodes * p.group + block - 1) / block : 0;
    }
#pragma unroll
    for (int o = 1; o < kWarp; o <<= 1) {
        const int up = __shfl_up_sync(0xFFFFFFFFu, units, o);
        if (lane >= o) units += up;
    }
    if (lane == kWarp - 1) warp_units[warp] = units;
    __syncthreads();
    for (int w = 0; w < warp; ++w) units += warp_units[w];
    unit_end[tid] = units;
    if (__syncthreads_or(gave_up)) {
        const long long cells = (long long)min(max(p.row_starts[p.batch], 0), p.rows) * p.q_heads * HD;
        for (long long i = (long long)blockIdx.x * kTreeMergeThreads + tid; i < cells; i += (long long)gridDim.x * kTreeMergeThreads)
            p.out[i] = 0x7FC0u;
        return;
    }
    const int total = unit_end[kTreeMergeThreads - 1];
    for (int u = blockIdx.x; u < total; u += gridDim.x) {
        int c = 0, hi = kTreeMergeThreads - 1;
        while (c < hi) {
            const int mid = (c + hi) >> 1;
            if (unit_end[mid] > u) hi = mid;
            else c = mid + 1;
        }
        const TreeSplit s = split_s[c];
        const bool few = s.parts <= kFew;
        const int block = few ? kWarp : kWarp / 4, step = few ? 1 : 4;
        const int i0 = (u - (c > 0 ? unit_end[c - 1] : 0)) * block;
        const int rows = s.nodes * p.group;
        const int i = min(i0 + lane % block, rows - 1);
        const int tile = i / (p.tile_nodes * p.group);
        const int r = tile * kTreeRows + i - tile * p.tile_nodes * p.group;
        auto slot_of = [&](int k) -> int { return k == 0 ? 2 * c + s.first_slot : 2 * (c + k); };
        float m = -INFINITY, l = 0.0f;
        float4 o[kCols];
#pragma unroll
        for (int j = 0; j < kCols; ++j) o[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        // o, l about m join o2, l2 about m2, the later part second.
        auto join = [&](float m2, float l2, const float4 (&o2)[kCols]) {
            const float to = fmaxf(m, m2);
            const float f = m == -INFINITY ? 0.0f : exp2f(m - to), f2 = m2 == -INFINITY ? 0.0f : exp2f(m2 - to);
            m = to;
            l = l * f + l2 * f2;
#pragma unroll
            for (int j = 0; j < kCols; ++j) {
                o[j].x = o[j].x * f + o2[j].x * f2;
                o[j].y = o[j].y * f + o2[j].y * f2;
                o[j].z = o[j].z * f + o2[j].z * f2;
                o[j].w = o[j].w * f + o2[j].w * f2;
            }
        };
#pragma unroll 4
        for (int k = lane / block; k < s.parts; k += step) {
            const int slot = slot_of(k);
            const float2 ml = p.part_ml[slot * 256 + r];
            float4 v[kCols];
#pragma unroll
            for (int j = 0; j < kCols; ++j) v[j] = p.part_o[((long long)slot * (HD / 4) + j * kTreeMergeWarps + warp) * 256 + r];
            join(ml.x, ml.y, v);
        }
        if (!few) {
#pragma unroll
            for (int x = 8; x < kWarp; x <<= 1) {
                const float m2 = __shfl_xor_sync(0xFFFFFFFFu, m, x), l2 = __shfl_xor_sync(0xFFFFFFFFu, l, x);
                float4 v[kCols];
#pragma unroll
                for (int j = 0; j < kCols; ++j) {
                    v[j].x = __shfl_xor_sync(0xFFFFFFFFu, o[j].x, x);
                    v[j].y = __shfl_xor_sync(0xFFFFFFFFu, o[j].y, x);
                    v[j].z = __shfl_xor_sync(0xFFFFFFFFu, o[j].z, x);
                    v[j].w = __shfl_xor_sync(0xFFFFFFFFu, o[j].w, x);
                }
                join(m2, l2, v);
            }
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        if (lane < block) {
#pragma unroll
            for (int j = 0; j < kCols; ++j) {
                block_s[lane][j * kTreeMergeWarps + warp] =
                    make_uint2(pack_bf16(o[j].x * inv, o[j].y * inv), pack_bf16(o[j].z * inv, o[j].w * inv));
            }
        }
        __syncthreads();
        for (int x = tid; x < block * (HD / 4); x += kTreeMergeThreads) {
            const int j = i0 + x / (HD / 4);
            if (j >= rows) break;
            const int n = j / p.group, h = j - n * p.group;
            *reinterpret_cast<uint2 *>(p.out + ((long long)(s.row0 + n) * p.q_heads + s.kvh * p.group + h) * HD + x % (HD / 4) * 4) =
                block_s[x / (HD / 4)][x % (HD / 4)];
        }
        __syncthreads();
    }
}

}  // namespace cheetah
