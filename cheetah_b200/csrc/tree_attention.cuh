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
// A CTA (12 warps; the last two idle):
//   warp 0     TMA producer: Q boxes [64 dims, group heads, nodes], K and V
//              tiles in boxes of up to 64 keys of one page, through a ring of
//              single K or V tiles in the order the MMAs use them;
//   warp 1     owns TMEM; lane 0 issues S = Q K^T (128 x 128) and O += P V for
//              jobs i = 0, 1, 2, ... of the groups i % 2: S(0), S(1), then
//              PV(i), S(i+2), so one group's products run during the other's
//              softmax;
//   warps 2-9  two softmax groups, one thread per row: read the S row from
//              TMEM, mask, exponentials, P as bf16 back into S's columns (the
//              A operand of PV is read from TMEM). The running maximum moves
//              only when it grows by more than 2^8 (P and l use the same one,
//              so the quotient is the same), and O is rescaled in TMEM only
//              then.
// P is rounded to bf16 because the tensor cores multiply bf16; sums,
// statistics and O stay f32.
//
// Cells that a row must not see never reach it: their scores are replaced
// before the softmax, and a tile that holds any (nodes, the end of the
// sequence, a window, a page outside the pool) has the V rows that hold no
// position zeroed in shared memory, where P = 0 times a stale NaN would not
// stay 0. A node's own non-finite V is zeroed there as well, and added to the
// rows that do see it after the products (patch_row).
//
// All mbarrier waits are bounded: on a timeout the CTA waits (bounded) for its
// own copies and MMAs in flight, frees its TMEM and exits.
#pragma once

#include "attention_mma.cuh"
#include "common.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace cheetah {

constexpr int kTreeKeys = 128;      // keys per tile
constexpr int kTreeRows = 128;      // rows of a Q tile
constexpr int kTreeThreads = 320;
constexpr int kTreeMinShare = 2;    // key tiles a CTA takes at least (one per softmax group)
constexpr float kTreeRescaleLog2 = 8.0f;
constexpr uint32_t kTreeOCol = 256; // S_A | S_B | O_A | O_B
constexpr int kTreeMergeThreads = 256;
constexpr int kTreeMergeSplit = 8;

template <int HD>
struct TreeCfg {
    static constexpr int kHalves = HD / 64;
    static constexpr int kHalfBytes = kTreeKeys * 128;   // 64 dimensions of a tile
    static constexpr int kTile = kTreeKeys * HD * 2;     // one K, V or Q tile
    static constexpr int kBufs = HD == 64 ? 12 : 5;      // ring
    static constexpr int kTiles = 2 * kTile + kBufs * kTile;
};

// What a split item needs to be joined, written by the CTA that begins it.
struct TreeSplit {
    int row0, nodes, kvh, two_tiles;
    int first_slot;  // of the beginning; the other parts are slot 0 of the next CTAs
    int parts;       // 0: nothing to join
    int pad[2];
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
    float *part_o;      // [CTAs][2][256][HD], unnormalised
    float2 *part_ml;    // [CTAs][2][256]
};

// A run of key tiles [t0, t1) of one item.
struct TreeSegment {
    int row0, n;           // the sequence's first row and row count
    int ctx, len;          // context keys; cached positions within the table
    int b, kvh;
    int node0, nodes;      // the item's nodes within the sequence
    int t0, t1, first_tile, last_tile;
    int jobs;              // MMA jobs of this segment (0: rows to be zeroed)
    bool two_tiles;
    int low;               // first key any row may see
};

// Rows, context and tile range of sequence b.
struct TreeSeq {
    int row0, n, ctx, len, tile_lo, tiles, row_items;
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeAttnParams &p, int b) {
    TreeSeq s;
    const int r0 = p.row_starts[b], r1 = p.row_starts[b + 1], len = p.seq_lens[b];
    s.row0 = min(max(r0, 0), p.rows);
    s.n = max(min(r1, p.rows) - s.row0, 0);
    s.ctx = len - s.n;
    s.len = (int)min((long long)len, (long long)p.max_pages * p.page_tokens);
    const int low = p.window > 0 ? max(0, s.ctx - p.window + 1) : 0;
    s.tile_lo = low / kTreeKeys;
    // Without room for its rows a sequence is one unit that writes zeros.
    s.tiles = s.ctx < 0 ? 1 : max(1, (s.len + kTreeKeys - 1) / kTreeKeys - s.tile_lo);
    s.row_items = (s.n + 2 * p.tile_nodes - 1) / (2 * p.tile_nodes);
    return s;
}
__device__ __forceinline__ long long tree_units(const TreeAttnParams &p, const TreeSeq &s) {
    return (long long)s.row_items * p.kv_heads * s.tiles;
}

// Walks the segments of one CTA's share of the unit axis.
struct TreeWalk {
    int b;
    long long off;   // units into sequence b
    long long left;  // units left in the share
    TreeSeq s;
    bool fresh;

    __device__ __forceinline__ void start(int b0, long long off0, long long count) {
        b = b0;
        off = off0;
        left = count;
        fresh = true;
    }
    __device__ __forceinline__ bool next(const TreeAttnParams &p, TreeSegment &g) {
        if (left <= 0) return false;
        while (true) {
            if (b >= p.batch) return false;
            if (fresh) {
                s = tree_seq(p, b);
                fresh = false;
            }
            if (off < tree_units(p, s)) break;
            off = 0;
            ++b;
            fresh = true;
        }
        const int item = (int)(off / s.tiles), at = (int)(off % s.tiles);
        const int take = (int)min(left, (long long)(s.tiles - at));
        off += take;
        left -= take;
        const int rt = item % s.row_items;
        g.row0 = s.row0;
        g.n = s.n;
        g.ctx = s.ctx;
        g.len = s.len;
        g.b = b;
        g.kvh = item / s.row_items;
        g.node0 = rt * 2 * p.tile_nodes;
        g.nodes = min(s.n - g.node0, 2 * p.tile_nodes);
        g.two_tiles = g.nodes > p.tile_nodes;
        g.first_tile = s.tile_lo;
        g.last_tile = s.tile_lo + s.tiles;
        g.t0 = s.tile_lo + at;
        g.t1 = g.t0 + take;
        g.jobs = s.ctx < 0 ? 0 : (g.two_tiles ? 2 * take : take);
        g.low = p.window > 0 ? max(0, s.ctx - p.window + 1) : 0;
        return true;
    }
};

// The ring position of tile i's K and V within a segment of T tiles, in the
// order of first use: K0 V0 K1 V1 .. where both groups use each tile, and
// K0 K1 V0 K2 V1 K3 .. where they alternate.
__device__ __forceinline__ int tree_pos_k(bool two, int i, int T) {
    return two ? 2 * i : (i < 2 ? i : 2 * i - 1);
}
__device__ __forceinline__ int tree_pos_v(bool two, int i, int T) {
    return two ? 2 * i + 1 : (T == 1 ? 1 : 2 + i + min(i, T - 2));
}

struct TreeShared {
    uint64_t full[12], empty[12];
    uint64_t q_full, q_empty, s_full[2], p_full[2], seg_done, exchange, drain;
    long long warp_sums[10];
    long long total, start_off, share;
    uint32_t tmem;
    int start_b, abort_flag, non_finite;
    uint32_t valid[12];  // per ring buffer: which 16-key parts hold loaded positions
    float2 ml[2][kTreeRows];
};

template <int HD>
constexpr size_t tree_attention_smem() { return (size_t)TreeCfg<HD>::kTiles + 3072; }
static_assert(sizeof(TreeShared) <= 3072 - 512, "fits behind the tiles");

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

// Adds the non-finite values of the V rows that `row` sees in [t0, t1) to the
// result this thread has just stored (columns d0 .. d0+cols). Their products
// were left out of the MMAs.
template <int HD>
__device__ __noinline__ void patch_row(const TreeAttnParams &p, const TreeSegment &g, int row, int d0, int cols,
                                       uint16_t *out, float *part) {
    const int begin = p.window > 0 ? g.t0 * kTreeKeys : max(g.t0 * kTreeKeys, g.ctx / kTreeKeys * kTreeKeys);
    for (int p0 = begin; p0 < min(g.t1 * kTreeKeys, g.len); p0 += 32) {
        for (uint32_t rest = tree_visible(p, g, row, p0); rest; rest &= rest - 1) {
            const int pos = p0 + __ffs(rest) - 1;
            const int page = p.page_table[(long long)g.b * p.max_pages + pos / p.page_tokens];
            if (page < 0 || page >= p.num_pages) continue;
            const uint16_t *v = p.v_pool + (((long long)page * p.kv_heads + g.kvh) * p.page_tokens + pos % p.page_tokens) * HD;
            for (int d = d0; d < d0 + cols; ++d) {
                if (!bf16_non_finite(v[d])) continue;
                if (part) part[d] += bf16_to_f32(v[d]);
                else out[d] = f32_to_bf16_rne(bf16_to_f32(out[d]) + bf16_to_f32(v[d]));
            }
        }
    }
}

template <int HD>
__global__ void __launch_bounds__(kTreeThreads, 1)
    tree_attention_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                          const __grid_constant__ CUtensorMap v_map, const TreeAttnParams p) {
    using C = TreeCfg<HD>;
    constexpr uint32_t kIdescS = umma_idesc_bf16(kTreeRows, kTreeKeys);
    constexpr uint32_t kIdescPV = umma_idesc_bf16(kTreeRows, HD) | (1u << 16);  // V MN-major
    extern __shared__ __align__(1024) uint8_t tree_smem[];
    // The kernel has no other shared memory, so the dynamic part begins at a
    // 1024-byte boundary; 512 bytes of slack are left all the same.
    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(tree_smem) + 1023) & ~uintptr_t(1023));
    uint8_t *q_s = base, *ring = base + 2 * C::kTile;
    TreeShared &sh = *reinterpret_cast<TreeShared *>(base + C::kTiles);
    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;

    if (threadIdx.x == 0) {
        for (int i = 0; i < C::kBufs; ++i) {
            mbar_init(smem_u32(&sh.full[i]), 1);
            mbar_init(smem_u32(&sh.empty[i]), 1);
        }
        mbar_init(smem_u32(&sh.q_full), 1);
        mbar_init(smem_u32(&sh.q_empty), 1);
        for (int g = 0; g < 2; ++g) {
            mbar_init(smem_u32(&sh.s_full[g]), 1);
            mbar_init(smem_u32(&sh.p_full[g]), 4);
        }
        mbar_init(smem_u32(&sh.seg_done), 1);
        mbar_init(smem_u32(&sh.exchange), 8);
        mbar_init(smem_u32(&sh.drain), 1);
        sh.abort_flag = 0;
        sh.non_finite = 0;
        sh.start_b = p.batch;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                     "r"(512u));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    pdl_wait();
    pdl_launch_dependents();

    // Total units, then the sequence in which this CTA's share begins.
    long long mine = 0;
    for (int b = threadIdx.x; b < p.batch; b += kTreeThreads) mine += tree_units(p, tree_seq(p, b));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xFFFFFFFFu, mine, o);
    if (lane == 0) sh.warp_sums[warp] = mine;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    long long total = 0;
    for (int w = 0; w < kTreeThreads / kWarp; ++w) total += sh.warp_sums[w];
    const long long share = max((long long)kTreeMinShare, (total + gridDim.x - 1) / gridDim.x);
    const long long u0 = blockIdx.x * share;
    long long before = 0;
    for (int b0 = 0; b0 < p.batch && u0 < total; b0 += kTreeThreads) {
        const int b = b0 + threadIdx.x;
        const long long units = b < p.batch ? tree_units(p, tree_seq(p, b)) : 0;
        long long v = units;
#pragma unroll
        for (int o = 1; o < kWarp; o <<= 1) {
            const long long up = __shfl_up_sync(0xFFFFFFFFu, v, o);
            if (lane >= o) v += up;
        }
        __syncthreads();
        if (lane == kWarp - 1) sh.warp_sums[warp] = v;
        __syncthreads();
        for (int w = 0; w < warp; ++w) v += sh.warp_sums[w];
        v += before;
        if (v - units <= u0 && u0 < v) {
            sh.start_b = b;
            sh.start_off = u0 - (v - units);
        }
        for (int w = 0; w < kTreeThreads / kWarp; ++w) before += sh.warp_sums[w];
    }
    __syncthreads();
    TreeWalk walk;
    walk.start(sh.start_b, sh.start_off, u0 < total ? min(share, total - u0) : 0);
    TreeSegment g;

    int ring_at = 0;       // ring positions of the segments before
    int issued = 0;        // producer: positions requested
    int q_issued = 0;
    if (warp == 0) {
        const int boxes = kTreeKeys / p.box_keys;
        const int parts = p.box_keys / 16;  // 16-key parts of a box
        int segs = 0;
        bool ok = true;
        while (ok && walk.next(p, g)) {
            if (g.jobs == 0) continue;
            const int T = g.t1 - g.t0;
            const int32_t *table = p.page_table + (long long)g.b * p.max_pages;
            // Page ids of 32 consecutive boxes, one per lane, for K and for V.
            int base_k = -1, base_v = -1, page_k = -1, page_v = -1;
            auto page_of = [&](int box, int &first, int &page) -> int {
                if (first < 0 || box < first || box >= first + kWarp) {
                    first = box;
                    const long long pos = (long long)(box + lane) * p.box_keys;
                    page = -1;
                    if (pos < g.len && pos + p.box_keys > g.low) {
                        const int id = table[(int)pos / p.page_tokens];
                        if (id >= 0 && id < p.num_pages) page = id;
                    }
                }
                return first;
            };
            for (int pos = 0; ok && pos < 2 * T; ++pos) {
                if (pos == min(2, 2 * T - 1)) {
                    // Q, once the previous segment's S products are done.
                    ok = __all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&sh.q_empty), (segs & 1) ^ 1));
                    if (!ok) break;
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
                    ++segs;
                }
                bool is_v;
                int i;
                if (g.two_tiles) {
                    i = pos >> 1;
                    is_v = pos & 1;
                } else if (T == 1 || pos < 2) {
                    i = T == 1 ? 0 : pos;
                    is_v = T == 1 && pos == 1;
                } else {
                    const int x = pos - 2, mixed = 2 * (T - 2);
                    is_v = x >= mixed || (x & 1) == 0;
                    i = x >= mixed ? T - 2 + (x - mixed) : (is_v ? x >> 1 : 2 + (x >> 1));
                }
                const int at = ring_at + pos;
                const int buf = at % C::kBufs;
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&sh.empty[buf]), ((at / C::kBufs) & 1) ^ 1));
                if (!ok) break;
                const int box0 = (g.t0 + i) * boxes;
                // A tile's boxes never straddle the 32 ids (32 is a multiple of 2, 4 and 8).
                const int first = is_v ? page_of(box0, base_v, page_v) : page_of(box0, base_k, page_k);
                const int box = lane % boxes, half = lane / boxes;
                const int page = __shfl_sync(0xFFFFFFFFu, is_v ? page_v : page_k, box0 + box - first);
                const uint32_t good = __ballot_sync(0xFFFFFFFFu, page >= 0) & low_bits(boxes);
                const uint32_t bar = smem_u32(&sh.full[buf]);
                if (lane == 0) {
                    uint32_t valid = 0;
                    for (int x = 0; x < boxes; ++x) {
                        if (good >> x & 1) valid |= low_bits(parts) << (x * parts);
                    }
                    sh.valid[buf] = valid;
                    mbar_expect_tx(bar, (uint32_t)(__popc(good) * p.box_keys * HD * 2));
                }
                __syncwarp();
                if (half < C::kHalves && page >= 0) {
                    const int key = (box0 + box) * p.box_keys;
                    const int row = (int)(((long long)page * p.kv_heads + g.kvh) * p.page_tokens + key % p.page_tokens);
                    tma_load_2d(smem_u32(ring + buf * C::kTile + half * C::kHalfBytes + box * p.box_keys * 128),
                                is_v ? &v_map : &k_map, half * 64, row, bar);
                }
                issued = at + 1;
            }
            ring_at += 2 * T;
        }
        if (!ok) sh.abort_flag = 1;
    } else if (warp == 1) {
        if (lane == 0) {
            int segs = 0;
            int seen[2] = {0, 0};  // P tiles consumed per group
            bool ok = true;
            while (ok && walk.next(p, g)) {
                if (g.jobs == 0) continue;
                const int T = g.t1 - g.t0;
                auto issue_s = [&](int i) -> bool {
                    const int grp = i & 1, tile = g.two_tiles ? i >> 1 : i;
                    const int at = ring_at + tree_pos_k(g.two_tiles, tile, T), buf = at % C::kBufs;
                    if (!mbar_wait(smem_u32(&sh.full[buf]), (at / C::kBufs) & 1)) return false;
                    tc_fence_after();
                    const uint32_t k_addr = smem_u32(ring + buf * C::kTile);
                    const uint32_t q_addr = smem_u32(q_s + (g.two_tiles ? grp * C::kTile : 0));
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k) {
                        const uint32_t off = (uint32_t)((k >> 2) * C::kHalfBytes + (k & 3) * 32);
                        umma_bf16(tmem + grp * kTreeKeys, umma_smem_desc(q_addr + off), umma_smem_desc(k_addr + off), kIdescS,
                                  k > 0 ? 1u : 0u);
                    }
                    umma_commit(smem_u32(&sh.s_full[grp]));
                    if (!g.two_tiles || grp == 1) umma_commit(smem_u32(&sh.empty[buf]));
                    if (i == g.jobs - 1) umma_commit(smem_u32(&sh.q_empty));
                    return true;
                };
                auto issue_pv = [&](int i) -> bool {
                    const int grp = i & 1, tile = g.two_tiles ? i >> 1 : i;
                    const int at = ring_at + tree_pos_v(g.two_tiles, tile, T), buf = at % C::kBufs;
                    if (!mbar_wait(smem_u32(&sh.p_full[grp]), seen[grp] & 1)) return false;
                    ++seen[grp];
                    if (!mbar_wait(smem_u32(&sh.full[buf]), (at / C::kBufs) & 1)) return false;
                    tc_fence_after();
                    const uint32_t v_addr = smem_u32(ring + buf * C::kTile);
#pragma unroll
                    for (int k = 0; k < kTreeKeys / 16; ++k) {
                        umma_bf16_ta(tmem + kTreeOCol + grp * HD, tmem + grp * kTreeKeys + k * 8,
                                     umma_smem_desc_mn(v_addr + k * 2048, HD > 64 ? C::kHalfBytes : 16), kIdescPV,
                                     (i > 1 || k > 0) ? 1u : 0u);
                    }
                    if (!g.two_tiles || grp == 1) umma_commit(smem_u32(&sh.empty[buf]));
                    if (i == g.jobs - 1) umma_commit(smem_u32(&sh.seg_done));
                    return true;
                };
                ok = mbar_wait(smem_u32(&sh.q_full), segs & 1);
                ++segs;
                if (ok) ok = issue_s(0) && (g.jobs < 2 || issue_s(1));
                for (int i = 0; ok && i < g.jobs; ++i) ok = issue_pv(i) && (i + 2 >= g.jobs || issue_s(i + 2));
                ring_at += 2 * T;
            }
            if (!ok) sh.abort_flag = 1;
        }
    } else {
        const int grp = (warp - 2) / 4, quad = warp % 4;
        const int r = quad * 32 + lane;
        const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
        const uint32_t s_addr = tmem + lane_off + grp * kTreeKeys;
        const uint32_t o_addr = tmem + lane_off + kTreeOCol + grp * HD;
        const int node_of_r = r / p.group, head_of_r = r % p.group;
        int done_s = 0, done_seg = 0, done_x = 0;
        bool ok = true, cut = false;
        int cut_first_slot = 0, cut_parts = 0;
        TreeSegment cut_seg;
        long long at_unit = u0;
        bool first_seg = true;
        while (ok && walk.next(p, g)) {
            const int T = g.t1 - g.t0;
            const int tile_grp = g.two_tiles ? grp : 0;
            const int node = g.node0 + tile_grp * p.tile_nodes + node_of_r;
            const bool live = node_of_r < p.tile_nodes && node < g.node0 + g.nodes;
            const int row = g.row0 + node;
            const int head = g.kvh * p.group + head_of_r;
            uint16_t *out_row = p.out + ((long long)row * p.q_heads + head) * HD;
            const bool whole = g.t0 == g.first_tile && g.t1 == g.last_tile;
            const int slot = first_seg ? 0 : 1;
            if (g.t0 == g.first_tile && !whole) {
                cut = true;
                cut_first_slot = slot;
                cut_seg = g;
                cut_parts = (int)((at_unit + (g.last_tile - g.first_tile) - 1) / share - blockIdx.x) + 1;
            }
            at_unit += T;
            first_seg = false;
            if (g.jobs == 0) {
                if (live && (g.two_tiles || grp == 0)) {
#pragma unroll
                    for (int i = 0; i < HD / 8; ++i) reinterpret_cast<uint4 *>(out_row)[i] = make_uint4(0u, 0u, 0u, 0u);
                }
                continue;
            }
            const bool warp_live = __any_sync(0xFFFFFFFFu, live);
            float m_run = -INFINITY, l_run = 0.0f;
            for (int i = grp; i < g.jobs; i += 2) {
                if (!__all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&sh.s_full[grp]), done_s & 1))) {
                    ok = false;
                    break;
                }
                ++done_s;
                const int tile = g.two_tiles ? i >> 1 : i;
                const int at = ring_at + tree_pos_v(g.two_tiles, tile, T), buf = at % C::kBufs;
                // V of this tile stays until this group's P is consumed, so
                // its phase cannot have moved on.
                if (!__all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&sh.full[buf]), (at / C::kBufs) & 1))) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const int p0 = (g.t0 + tile) * kTreeKeys;
                const uint32_t valid = sh.valid[buf];
                const bool masked = p.window > 0 || p0 + kTreeKeys > g.ctx || valid != 0xFFu;
                uint32_t vis[4] = {0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu};
                if (masked) {
                    // V row r: zero where no position is, finite elsewhere.
                    uint8_t *v_row = ring + buf * C::kTile + r * 128;
                    const bool holds = p0 + r < g.len && (valid >> (r >> 4) & 1);
#pragma unroll 1
                    for (int c = 0; c < HD / 8; ++c) {
                        uint4 *cell = reinterpret_cast<uint4 *>(v_row + (c >> 3) * C::kHalfBytes + (c & 7) * 16);
                        if (!holds) {
                            *cell = make_uint4(0u, 0u, 0u, 0u);
                            continue;
                        }
                        uint32_t w[4] = {cell->x, cell->y, cell->z, cell->w};
                        bool bad = false;
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            if (bf16_non_finite(w[x])) {
                                w[x] &= 0xFFFF0000u;
                                bad = true;
                            }
                            if (bf16_non_finite(w[x] >> 16)) {
                                w[x] &= 0x0000FFFFu;
                                bad = true;
                            }
                        }
                        if (bad) {
                            *reinterpret_cast<volatile int *>(&sh.non_finite) = 1;
                            __threadfence_block();  // flag before the zeros that hide it from the other group
                            *cell = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const uint32_t part = (valid >> (2 * c) & 1 ? 0x0000FFFFu : 0u) | (valid >> (2 * c + 1) & 1 ? 0xFFFF0000u : 0u);
                        vis[c] = live ? tree_visible(p, g, row, p0 + 32 * c) & part : 0u;
                    }
                }
                if (warp_live) {
                    float mx[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) mx[k] = -INFINITY;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float sc[64];
                        tmem_ld32_nowait(s_addr + h * 64, sc);
                        tmem_ld32_nowait(s_addr + h * 64 + 32, sc + 32);
                        tmem_wait_ld();
                        if (masked) {
#pragma unroll
                            for (int k = 0; k < 64; ++k) sc[k] = (vis[2 * h + (k >> 5)] >> (k & 31) & 1) ? sc[k] : -INFINITY;
                        }
#pragma unroll
                        for (int k = 0; k < 64; ++k) mx[k & 7] = fmaxf(mx[k & 7], sc[k]);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) mx[k] = fmaxf(mx[k], mx[k + 4]);
                    const float tmax = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;
                    const float m_cand = fmaxf(m_run, tmax);
                    const float m_new = m_cand > m_run + kTreeRescaleLog2 ? m_cand : m_run;
                    const float alpha = m_new == -INFINITY ? 1.0f : exp2f(m_run - m_new);
                    const float neg_m = m_new == -INFINITY ? 0.0f : -m_new;
                    if (i > 1 && __any_sync(0xFFFFFFFFu, alpha < 1.0f)) {
#pragma unroll 1
                        for (int c = 0; c < HD / 32; ++c) {
                            float ov[32];
                            tmem_ld32(o_addr + c * 32, ov);
#pragma unroll
                            for (int k = 0; k < 32; ++k) ov[k] *= alpha;
                            tmem_st32(o_addr + c * 32, ov);
                        }
                    }
                    float sums[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) sums[k] = 0.0f;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float sc[64];
                        tmem_ld32_nowait(s_addr + h * 64, sc);
                        tmem_ld32_nowait(s_addr + h * 64 + 32, sc + 32);
                        tmem_wait_ld();
                        if (masked) {
#pragma unroll
                            for (int k = 0; k < 64; ++k) sc[k] = (vis[2 * h + (k >> 5)] >> (k & 31) & 1) ? sc[k] : -INFINITY;
                        }
                        uint32_t w[32];
#pragma unroll
                        for (int k = 0; k < 32; ++k) {
                            const float e0 = fast_exp2(fmaf(sc[2 * k], p.scale_log2, neg_m));
                            const float e1 = fast_exp2(fmaf(sc[2 * k + 1], p.scale_log2, neg_m));
                            sums[k & 7] += e0 + e1;
                            w[k] = pack_bf16(e0, e1);
                        }
                        // P columns 32h..32h+31: S columns already read.
                        tmem_st32_nowait(s_addr + h * 32, w);
                    }
                    tmem_wait_st();
#pragma unroll
                    for (int k = 0; k < 4; ++k) sums[k] += sums[k + 4];
                    l_run = l_run * alpha + ((sums[0] + sums[1]) + (sums[2] + sums[3]));
                    m_run = m_new;
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.p_full[grp]));
            }
            ring_at += 2 * T;
            if (!ok) break;
            if (!__all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&sh.seg_done), done_seg & 1))) {
                ok = false;
                break;
            }
            ++done_seg;
            tc_fence_after();
            // Weights of this row's accumulators: its own, and the other
            // group's where both hold the same row.
            float w_own = 1.0f, w_other = 0.0f, l = l_run, m = m_run;
            int d0 = 0, cols = HD;
            if (!g.two_tiles) {
                sh.ml[grp][r] = make_float2(m_run, l_run);
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.exchange));
                if (!__all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&sh.exchange), done_x & 1))) {
                    ok = false;
                    break;
                }
                ++done_x;
                const float2 other = sh.ml[grp ^ 1][r];
                m = fmaxf(m_run, other.x);
                w_own = m_run == -INFINITY ? 0.0f : exp2f(m_run - m);
                w_other = other.x == -INFINITY ? 0.0f : exp2f(other.x - m);
                l = l_run * w_own + other.y * w_other;
                // Group A finishes the first half of the columns, B the second.
                d0 = grp * (HD / 2);
                cols = HD / 2;
            }
            const bool joined = !g.two_tiles && g.jobs > 1;
            const uint32_t own = o_addr, other_addr = tmem + lane_off + kTreeOCol + (grp ^ 1) * HD;
            // Where one tile was all, only group A has accumulated.
            const uint32_t only = tmem + lane_off + kTreeOCol;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            const long long part_row = (long long)(2 * blockIdx.x + slot) * 256 + tile_grp * kTreeRows + r;
            float *part = p.part_o + part_row * HD;
            if (warp_live) {
#pragma unroll 1
                for (int c = d0; c < d0 + cols; c += 32) {
                    float ov[32];
                    if (joined) {
                        float ox[32];
                        tmem_ld32_nowait(own + c, ov);
                        tmem_ld32_nowait(other_addr + c, ox);
                        tmem_wait_ld();
#pragma unroll
                        for (int k = 0; k < 32; ++k) ov[k] = ov[k] * w_own + ox[k] * w_other;
                    } else {
                        tmem_ld32(g.two_tiles ? own + c : only + c, ov);
                    }
                    if (!live) continue;
                    if (whole) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            reinterpret_cast<uint4 *>(out_row + c)[k] =
                                make_uint4(pack_bf16(ov[8 * k] * inv, ov[8 * k + 1] * inv), pack_bf16(ov[8 * k + 2] * inv, ov[8 * k + 3] * inv),
                                           pack_bf16(ov[8 * k + 4] * inv, ov[8 * k + 5] * inv), pack_bf16(ov[8 * k + 6] * inv, ov[8 * k + 7] * inv));
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            reinterpret_cast<float4 *>(part + c)[k] = make_float4(ov[4 * k], ov[4 * k + 1], ov[4 * k + 2], ov[4 * k + 3]);
                    }
                }
                if (live) {
                    if (!whole && (g.two_tiles || grp == 0)) p.part_ml[part_row] = make_float2(m, l);
                    if (*reinterpret_cast<volatile int *>(&sh.non_finite))
                        patch_row<HD>(p, g, row, d0, cols, out_row, whole ? nullptr : part);
                }
            }
            tc_fence_before();
            // Neither accumulator may be overwritten before both are read, and
            // neither group may fall a segment behind the other's barriers.
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.exchange));
            if (!__all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&sh.exchange), done_x & 1))) {
                ok = false;
                break;
            }
            ++done_x;
        }
        if (!ok) sh.abort_flag = 1;
        if (threadIdx.x == 2 * kWarp) {
            TreeSplit s = {};
            if (cut) {
                s.row0 = cut_seg.row0 + cut_seg.node0;
                s.nodes = cut_seg.nodes;
                s.kvh = cut_seg.kvh;
                s.two_tiles = cut_seg.two_tiles;
                s.first_slot = cut_first_slot;
                s.parts = cut_parts;
            }
            p.splits[blockIdx.x] = s;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (sh.abort_flag) {
        // A wait gave up: let this CTA's copies and MMAs still in flight land
        // before its shared memory and TMEM are released (bounded waits).
        if (warp == 0 && lane == 0) {
            if (q_issued > 0) mbar_wait(smem_u32(&sh.q_full), (q_issued - 1) & 1);
            for (int at = max(0, issued - C::kBufs); at < issued; ++at)
                mbar_wait(smem_u32(&sh.full[at % C::kBufs]), (at / C::kBufs) & 1);
        } else if (warp == 1 && lane == 0) {
            umma_commit(smem_u32(&sh.drain));
            mbar_wait(smem_u32(&sh.drain), 0);
        }
        tc_fence_before();
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
    }
}

// Joins the parts of the items that shares cut: o = sum_k 2^(m_k - m) o_k /
// sum_k 2^(m_k - m) l_k, parts in key order. CTA (x, y): the item that CTA x
// began, every kTreeMergeSplit-th block of its rows; HD/4 lanes per row.
template <int HD>
__global__ void __launch_bounds__(kTreeMergeThreads) tree_merge_kernel(const TreeAttnParams p) {
    constexpr int kLanes = HD / 4;
    constexpr int kRowsPerCta = kTreeMergeThreads / kLanes;
    pdl_wait();
    pdl_launch_dependents();
    const TreeSplit s = p.splits[blockIdx.x];
    if (s.parts < 2) return;
    const int lane = threadIdx.x % kLanes;
    const int first = 2 * blockIdx.x + s.first_slot;
    for (int i = blockIdx.y * kRowsPerCta + threadIdx.x / kLanes; i < s.nodes * p.group; i += kTreeMergeSplit * kRowsPerCta) {
        const int node = i / p.group, head = i % p.group;
        const int tile = node / p.tile_nodes;
        const int r = tile * kTreeRows + (node - tile * p.tile_nodes) * p.group + head;
        auto part_at = [&](int k) -> long long { return (long long)(k == 0 ? first : 2 * (blockIdx.x + k)) * 256 + r; };
        float m = -INFINITY;
        for (int k = 0; k < s.parts; ++k) m = fmaxf(m, p.part_ml[part_at(k)].x);
        float l = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int k = 0; k < s.parts; ++k) {
            const long long at = part_at(k);
            const float2 ml = p.part_ml[at];
            const float4 v = *reinterpret_cast<const float4 *>(p.part_o + at * HD + lane * 4);
            const float w = ml.x == -INFINITY ? 0.0f : exp2f(ml.x - m);
            l = fmaf(ml.y, w, l);
            o.x = fmaf(v.x, w, o.x);
            o.y = fmaf(v.y, w, o.y);
            o.z = fmaf(v.z, w, o.z);
            o.w = fmaf(v.w, w, o.w);
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        *reinterpret_cast<uint2 *>(p.out + ((long long)(s.row0 + node) * p.q_heads + s.kvh * p.group + head) * HD + lane * 4) =
            make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
    }
}

}  // namespace cheetah
