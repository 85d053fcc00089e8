// Causal attention of a batch's new rows over an 8-bit paged cache: what its
// kernels share.
//
//   o_i = sum_j softmax_j(q_i . k_j / sqrt(D)) v_j,   k_j = kc_j ks,  v_j = vc_j vs
//
// with e4m3 codes and one scale per 16 cells and head, in one pass over the keys
// with a running reference m and sum (log2 units, t_j = log2(e)/sqrt(D) q . k_j):
//   w_j = 2^(t_j + log2(vs) - m),   o' = sum_j w_j vc_j,   l = sum_j w_j / vs,   o = o' / l.
//
// The codes are multiplied as they are (tcgen05 kind::f8f6f4). What meets them
// is split into 8-bit parts that are multiplied one after the other: q, over a
// power of two of its row that puts the largest element at 224 or above, into two of
// e4m3 (exact for elements within 2^-10 of the row's largest, else off by half the
// smallest step, 2^-10 / 224 = 2^-17.8 of that); the weights times V's scale, through
// f16, into three of e5m2: off by 2^-9 + 2^-11 of themselves (bf16 holds 2^-8), or by
// half the smallest step, 2^-29 of the row's largest. That floor is what a tail of many
// small weights behind a heavy key needs: what is lost adds up over the keys,
// while l counts every weight in full. Two e4m3 parts, whose floor is 2^-16 of the largest,
// lost a third of such rows over 32768 keys; two of e5m2 hold 2^-6. K's scale joins
// the factor of the scores. m follows t_j + log2(vs), so the weights fill e5m2's
// range however V's scales differ.
//
// Work. An item is a run of rows of one (sequence, KV head): nodes (new tokens)
// times the query heads of the group, so K and V are read once for all of them.
// Its key tiles (128 keys) are those of the first `sinks` positions and from the
// window's begin to its last row's position. The tiles of all items lie on one
// axis that is cut into equal shares, one per CTA, one CTA per SM: ragged
// batches and a single long sequence fill the GPU alike. An item cut by a share's
// end leaves partial (o, m, l) in the workspace, and the merge joins them,
// always in the same order.
//
// Cells that a row must not see never reach it: their weights are 0, and a V cell
// that holds no position, or a NaN that some row does not see, is zeroed in shared
// memory first, where 0 times NaN would not stay 0; the rows that do see it are
// made NaN at the end (kv8_patch).
//
// Shares, splits of items and the list of parts are those of tree_attention.cuh.
//
// All mbarrier waits are bounded: on a timeout the CTA waits (bounded) for its
// own copies and MMAs in flight, frees its TMEM and exits, and the merge makes
// every row NaN.
#pragma once

#include <limits.h>

#include "common.cuh"
#include "kv8.cuh"
#include "pair.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"
#include "tree_attention.cuh"

namespace cheetah {

constexpr int kKv8Keys = 128;     // keys per tile
constexpr int kKv8MaxCtas = kTreeMaxCtas;
constexpr int kKv8Queue = 4;      // segments the scheduler may be ahead
// Weights are scaled to at most 2^kKv8TopLog2 when a row's reference is set, and it
// moves when one would pass 2^kKv8RoomLog2 times that (e5m2 ends at 57344 = 2^15.8). A
// move costs a pass over O, and in 32 rows one moves soon; but what the room takes the
// floor loses. Prompts of 2 x 2000 rows took 318 us with 14 and 1.75, 317 with these,
// 315 with 12 and 3.75.
constexpr float kKv8TopLog2 = 13.0f, kKv8RoomLog2 = 2.75f;
constexpr int kKv8Parts = 3;      // of a weight

struct Kv8AttnParams {
    const uint16_t *q;
    long long q_stride;
    const uint8_t *k_codes, *v_codes;
    const float *k_scales, *v_scales;
    const int32_t *page_table;
    int max_pages, num_pages, page_tokens;
    int box_shift;     // log2 of the keys of a TMA box: 4 .. 7
    const int32_t *seq_lens, *row_starts;
    int batch, rows, window, sinks;
    int q_heads, kv_heads, group;
    int item_nodes;    // new tokens of an item at most
    int tile_nodes;    // and of one of its row tiles (few rows: the item's)
    float scale_log2;
    uint16_t *out;
    TreeSplit *splits;  // [CTAs]
    float *part_o;     // [CTAs][2][rows of an item][HD] unnormalised
    float2 *part_ml;   // [CTAs][2][rows of an item]
};

// A run of tiles [t0, t1) of one item.
struct Kv8Segment {
    int row0, nodes;    // the item's rows of q
    int pos0;           // position of the first
    int len;            // cached positions within the table
    int b, kvh;
    int t0, t1;
    int sink_tiles, skip;  // tile t >= sink_tiles covers the keys of tile t + skip
    int low;            // the first key that its first row sees in the window
    int jobs;           // tiles (0: rows to be zeroed; -1: no more segments)
    int slot;           // workspace slot of a part; -1: the segment is its whole item
    __device__ __forceinline__ int key0(int t) const { return (t < sink_tiles ? t : t + skip) * kKv8Keys; }
};

struct Kv8Seq {
    int row0, n, ctx, len, items;
};
__device__ __forceinline__ Kv8Seq kv8_seq(const Kv8AttnParams &p, int b) {
    Kv8Seq s;
    const int r0 = p.row_starts[b], r1 = p.row_starts[b + 1], len = p.seq_lens[b];
    s.row0 = min(max(r0, 0), p.rows);
    s.n = max(min(r1, p.rows) - s.row0, 0);
    s.ctx = len - s.n;
    s.len = (int)min((long long)len, (long long)p.max_pages * p.page_tokens);
    s.items = (s.n + p.item_nodes - 1) / p.item_nodes;
    return s;
}
// Tiles of item j of a sequence.
struct Kv8Range {
    int tiles, sink_tiles, skip, low;
};
__device__ __forceinline__ Kv8Range kv8_range(const Kv8AttnParams &p, const Kv8Seq &s, int j) {
    Kv8Range r = {1, 0, 0, 0};
    if (s.ctx < 0) return r;  // without room for its rows: one tile that writes zeros
    const int node0 = j * p.item_nodes, nodes = min(s.n - node0, p.item_nodes);
    r.low = p.window > 0 ? max(0, s.ctx + node0 - p.window + 1) : 0;
    // Up to the last row, within the table (a window may begin behind it).
    const int hi = (min(s.ctx + node0 + nodes, s.len) + kKv8Keys - 1) / kKv8Keys, lo = min(r.low / kKv8Keys, hi);
    r.sink_tiles = min((p.sinks + (kKv8Keys - 1LL)) / kKv8Keys, (long long)lo);
    r.skip = lo - r.sink_tiles;
    r.tiles = max(1, r.sink_tiles + hi - lo);
    return r;
}
// Cost units of a kernel: ITEM for an item's beginning and end, ONE or TWO for a
// key tile, by its row tiles. A share holds MIN_SHARE at least, which hold a tile.
template <int ITEM_, int ONE, int TWO, int MIN_SHARE_>
struct Kv8Cost {
    static constexpr int ITEM = ITEM_, TWO_TILES = TWO, MIN_SHARE = MIN_SHARE_;
    static_assert(MIN_SHARE >= TWO && TWO >= ONE, "every share holds a tile");
    static __device__ __forceinline__ int tile(const Kv8AttnParams &p, const Kv8Seq &s, int j) {
        return s.n - j * p.item_nodes > p.tile_nodes ? TWO : ONE;
    }
    static __device__ __forceinline__ int item(const Kv8AttnParams &p, const Kv8Seq &s, int j) {
        return ITEM + kv8_range(p, s, j).tiles * tile(p, s, j);
    }
    // Of one KV head of a sequence.
    static __device__ __forceinline__ int head(const Kv8AttnParams &p, const Kv8Seq &s) {
        int units = 0;
        for (int j = 0; j < s.items; ++j) units += item(p, s, j);
        return units;
    }
};

// The share of this CTA, segment by segment. Called by a whole warp, whose lanes
// then hold the same state.
template <typename Cost>
struct Kv8Walk {
    int b, j, kvh, left, unit, at, share, count;
    Kv8Seq s;
    TreeSplit split;

    __device__ __forceinline__ void init(const Kv8AttnParams &p) {
        // A lane per sequence; the units of the first kKept * 32 stay in registers. (Loads
        // side by side, the rest in loops that pass the registers on: this code runs once
        // and is the faster for being short.)
        constexpr int kKept = 4;
        const int lane = threadIdx.x % kWarp;
        auto units_of = [&](int i) -> int { return i < p.batch ? Cost::head(p, kv8_seq(p, i)) * p.kv_heads : 0; };
        int kept[kKept] = {}, total = 0;
        Kv8Seq first[kKept];
#pragma unroll
        for (int k = 0; k < kKept; ++k) first[k] = kv8_seq(p, min(lane + k * kWarp, p.batch - 1));
#pragma unroll 1
        for (int k = 0; k < kKept; ++k) {
            const int units = lane + k * kWarp < p.batch ? Cost::head(p, first[0]) * p.kv_heads : 0;
            total += units;
#pragma unroll
            for (int i = 0; i + 1 < kKept; ++i) {
                first[i] = first[i + 1];
                kept[i] = kept[i + 1];
            }
            kept[kKept - 1] = units;
        }
#pragma unroll 1
        for (int i = lane + kKept * kWarp; i < p.batch; i += kWarp) total += units_of(i);
        total = __reduce_add_sync(0xFFFFFFFFu, total);
        share = max(Cost::MIN_SHARE, (int)(((unsigned)total + gridDim.x - 1) / gridDim.x));
        const int u0 = (int)min((long long)blockIdx.x * share, (long long)total);
        int start = -1, before = 0;
        at = 0;
        auto look = [&](int b0, int units) {
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
        };
        if (u0 < total) {
#pragma unroll 1
            for (int b0 = 0; b0 < p.batch && start < 0; b0 += kWarp) {
                look(b0, b0 < kKept * kWarp ? kept[0] : units_of(b0 + lane));
#pragma unroll
                for (int i = 0; i + 1 < kKept; ++i) kept[i] = kept[i + 1];
            }
        }
        b = start;
        left = min(share, total - u0);
        unit = u0;
        j = kvh = count = 0;
        split = TreeSplit{};
        if (left > 0) {
            s = kv8_seq(p, b);
            const int head = Cost::head(p, s);
            kvh = at / head;
            at -= kvh * head;
            while (true) {
                const int units = Cost::item(p, s, j);
                if (at < units) break;
                at -= units;
                ++j;
            }
        }
    }
    __device__ __forceinline__ Kv8Segment next(const Kv8AttnParams &p) {
        Kv8Segment g = {};
        g.jobs = -1;
        while (left > 0) {
            const Kv8Range r = kv8_range(p, s, j);
            const int cost = Cost::tile(p, s, j), units = Cost::ITEM + r.tiles * cost;
            const int take = min(left, units - at);
            // Tiles of this piece; an item's first ITEM units hold none.
            const int t0 = max(at - Cost::ITEM, 0) / cost, t1 = max(at + take - Cost::ITEM, 0) / cost;
            if (t1 > t0) {
                const bool whole = t1 - t0 == r.tiles;
                const int node0 = j * p.item_nodes;
                g.row0 = s.row0 + node0;
                g.nodes = min(s.n - node0, p.item_nodes);
                g.pos0 = s.ctx + node0;
                g.len = s.len;
                g.b = b;
                g.kvh = kvh;
                g.t0 = t0;
                g.t1 = t1;
                g.sink_tiles = r.sink_tiles;
                g.skip = r.skip;
                g.low = r.low;
                g.jobs = s.ctx < 0 ? 0 : t1 - t0;
                g.slot = whole ? -1 : (count == 0 ? 0 : 1);
                if (t0 == 0 && !whole) {
                    split.row0 = g.row0;
                    split.nodes = g.nodes;
                    split.kvh = kvh;
                    split.first_slot = g.slot;
                    // Within the grid even if sequences share rows, which the units do not count on.
                    split.parts = min((unit - at + units - 1) / share - (int)blockIdx.x + 1, (int)(gridDim.x - blockIdx.x));
                }
                ++count;
            }
            unit += take;
            left -= take;
            at += take;
            if (at == units) {
                at = 0;
                if (++j == s.items) {
                    j = 0;
                    ++kvh;
                }
                while (left > 0 && kvh >= (s.items > 0 ? p.kv_heads : 0)) {  // the next sequence with rows
                    if (++b >= p.batch) {
                        left = 0;
                        break;
                    }
                    s = kv8_seq(p, b);
                    kvh = 0;
                }
            }
            if (t1 > t0) break;
        }
        return g;
    }
};

__device__ __forceinline__ uint32_t kv8_low_bits(int n) { return n <= 0 ? 0u : (n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u); }

// The pool rows of a segment's boxes (runs of 2^box_shift keys on one page), 32 of
// them at a time, one per lane; -1: not loaded. A tile's boxes never straddle
// the 32 (a multiple of 1, 2, 4 and 8).
struct Kv8Boxes {
    int first, row;
    __device__ __forceinline__ void reach(const Kv8AttnParams &p, const Kv8Segment &g, int box0) {
        if (box0 >= first && box0 < first + kWarp) return;
        first = box0;
        row = -1;
        const long long pos = (long long)(box0 + (int)(threadIdx.x % kWarp)) << p.box_shift;
        if (pos < min(g.len, g.pos0 + g.nodes) && (pos + (1 << p.box_shift) > g.low || pos < p.sinks)) {
            const int col = (int)pos / p.page_tokens;
            const int page = p.page_table[(long long)g.b * p.max_pages + col];
            if (page >= 0 && page < p.num_pages) row = (page * p.kv_heads + g.kvh) * p.page_tokens + ((int)pos - col * p.page_tokens);
        }
    }
};

// 16 bf16 elements of q (of a row that HD / 16 neighbouring lanes hold) as two e4m3
// parts of x / scale; the scale is a power of two of the row's largest element. All
// lanes of a warp call.
template <int HD>
__device__ __forceinline__ float kv8_split_q(const uint4 (&raw)[2], uint4 &part_hi, uint4 &part_lo) {
    constexpr int kCells = HD / 16;
    float x[16];
    const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[2 * i] = bf16_lo(w[i]);
        x[2 * i + 1] = bf16_hi(w[i]);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        if (fabsf(x[i]) < INFINITY) top = fmaxf(top, fabsf(x[i]));
        else x[i] = NAN;  // an infinity has no code
    }
#pragma unroll
    for (int o = kCells / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    const float scale = kv8_scale_for(__float_as_uint(top)), inv = 1.0f / scale;
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float v[4], h[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = x[4 * i + k] * inv;
        hi[i] = pack_e4m3x4(v[0], v[1], v[2], v[3]);
        unpack_e4m3x4(hi[i], h);
        lo[i] = pack_e4m3x4(v[0] - h[0], v[1] - h[1], v[2] - h[2], v[3] - h[3]);
    }
    part_hi = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    part_lo = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    return scale;
}

// The same for one row by a whole warp, a lane with HD / 32 elements; `src` is the
// row of q, or nullptr for zeros.
template <int HD>
__device__ __forceinline__ float kv8_split_row(const uint16_t *src, uint8_t *tile, int row, int row_lo) {
    constexpr int V = HD / kWarp;  // 4 or 2
    const int lane = threadIdx.x % kWarp;
    uint32_t w[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) w[i] = 0u;
    if (src != nullptr) {
        if constexpr (V == 4) {
            const uint2 raw = __ldg(reinterpret_cast<const uint2 *>(src) + lane);
            w[0] = raw.x;
            w[1] = raw.y;
        } else {
            w[0] = __ldg(reinterpret_cast<const uint32_t *>(src) + lane);
        }
    }
    float x[V];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        x[i] = i % 2 == 0 ? bf16_lo(w[i / 2]) : bf16_hi(w[i / 2]);
        const uint32_t mag = __float_as_uint(x[i]) & 0x7FFFFFFFu;
        if (mag < 0x7F800000u) top = max(top, mag);
        else x[i] = NAN;  // an infinity has no code
    }
    const float scale = kv8_scale_for(__reduce_max_sync(0xFFFFFFFFu, top));
    const float inv = __uint_as_float((254u << 23) - __float_as_uint(scale));  // of a power of two
    uint32_t hi[V / 2], lo[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
        const float a = x[2 * i] * inv, b = x[2 * i + 1] * inv;
        hi[i] = pack_e4m3x2(a, b);
        float ha, hb;
        unpack_e4m3x2(hi[i], ha, hb);
        lo[i] = pack_e4m3x2(a - ha, b - hb);
    }
    const int at = lane * V % 16, c = lane * V / 16;
    uint8_t *dst = tile + e4m3_tile_offset<HD>(row, c) + at, *dst_lo = tile + e4m3_tile_offset<HD>(row_lo, c) + at;
    if constexpr (V == 4) {
        *reinterpret_cast<uint32_t *>(dst) = hi[0] | hi[1] << 16;
        *reinterpret_cast<uint32_t *>(dst_lo) = lo[0] | lo[1] << 16;
    } else {
        *reinterpret_cast<uint16_t *>(dst) = (uint16_t)hi[0];
        *reinterpret_cast<uint16_t *>(dst_lo) = (uint16_t)lo[0];
    }
    return scale;
}

__device__ __forceinline__ void st_shared_u8(uint32_t addr, uint32_t v) { asm volatile("st.shared.u8 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }

__device__ __forceinline__ float kv8_log2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A producer warp's part of a segment: its K tiles, or its V tiles and the scales of
// both, into a ring of tiles `step` bytes apart. The scales go with V, whose stage is
// free only once the weights that need them are multiplied. False if a wait gave up.
template <int HD, int STAGES, bool IS_V>
__device__ __forceinline__ bool kv8_load_tiles(const Kv8AttnParams &p, const Kv8Segment &g, const CUtensorMap *map, uint64_t *full,
                                               uint64_t *empty, uint8_t *ring, int step, float (*scales)[16], uint32_t *valid_of,
                                               int tile_at, int &issued) {
    const int lane = threadIdx.x % kWarp, shift = p.box_shift, boxes = kKv8Keys >> shift;
    const uint32_t box_bytes = (uint32_t)HD << shift;
    // Scales: lanes 0..7 K's of a block each, 8..15 V's; `x` is the block's box.
    const int block = lane & 7, x = block >> (shift - 4), in_box = block & ((1 << (shift - 4)) - 1);
    const float *scale_of = lane < 8 ? p.k_scales : p.v_scales;
    Kv8Boxes box;
    box.first = INT_MIN / 2;
    box.row = -1;
    int buf = tile_at % STAGES, box0 = 0, row = -1;
    uint32_t phase = (tile_at / STAGES) & 1, valid = 0;
    float scale = 0.0f;
    // The next tile's boxes, and this lane's scale of it, on its way while others wait.
    auto look = [&](int t) {
        box0 = g.key0(t) >> shift;
        box.reach(p, g, box0);
        row = __shfl_sync(0xFFFFFFFFu, box.row, (box0 - box.first + x) & 31);  // of this lane's block
        valid = __ballot_sync(0xFFFFFFFFu, row >= 0) & 0xFFu;
        if (IS_V && lane < 16 && row >= 0) scale = __ldg(scale_of + row / kKv8Block + in_box);
    };
    const int t1 = g.t0 + g.jobs;
    if (g.jobs > 0) look(g.t0);
    for (int t = g.t0; t < t1; ++t) {
        if (!__all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&empty[buf]), phase ^ 1))) return false;
        const uint32_t bar = smem_u32(&full[buf]);
        // (The phase ends with the arrival below: it waits for these bytes as well.)
        const uint32_t dst = smem_u32(ring + buf * step);
        for (int i = 0; i < boxes; ++i) {
            const int box_row = __shfl_sync(0xFFFFFFFFu, box.row, box0 - box.first + i);
            if (lane == 0 && box_row >= 0) tma_load_2d(dst + i * box_bytes, map, 0, box_row, bar);
        }
        if (IS_V) {
            if (lane < 16) scales[buf][lane] = scale;
            if (lane == 0) valid_of[buf] = valid;
            __syncwarp();
        }
        if (lane == 0) mbar_expect_tx(bar, (uint32_t)__popc(valid) * kKv8Block * HD);
        __syncwarp();
        ++issued;
        if (++buf == STAGES) {
            buf = 0;
            phase ^= 1;
        }
        if (t + 1 < t1) look(t + 1);
    }
    return true;
}

// Whether a word holds a NaN code.
__device__ __forceinline__ uint32_t e4m3_nan_bits(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }

// One V row of a tile in shared memory: zero where it holds no position, else
// its NaN codes zeroed and noted for kv8_patch.
template <int HD>
__device__ __forceinline__ void kv8_clean_v(uint8_t *v_row, bool holds, int *non_finite) {
    constexpr int kCells = HD / 16;
    // Each lane begins at another cell: the rows lie 64 or 128 bytes apart.
    auto cell = [&](int c) -> uint4 & { return *reinterpret_cast<uint4 *>(v_row + ((c + threadIdx.x) % kCells) * 16); };
    if (!holds) {
#pragma unroll
        for (int c = 0; c < kCells; ++c) cell(c) = make_uint4(0u, 0u, 0u, 0u);
    } else {
        uint32_t bad = 0;
#pragma unroll
        for (int c = 0; c < kCells; ++c) {
            const uint4 v = cell(c);
            bad |= e4m3_nan_bits(v.x) | e4m3_nan_bits(v.y) | e4m3_nan_bits(v.z) | e4m3_nan_bits(v.w);
        }
        if (!bad) return;
        *reinterpret_cast<volatile int *>(non_finite) = 1;
        __threadfence_block();  // flag before the zeros that hide it from other warps
#pragma unroll 1
        for (int c = 0; c < kCells; ++c) {
            const uint4 v = cell(c);
            uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int x = 0; x < 4; ++x) w[x] &= ~((e4m3_nan_bits(w[x]) >> 7) * 0xFFu);
            cell(c) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

// Whether a row at `pos` sees key j (pages aside).
__device__ __forceinline__ bool kv8_sees(const Kv8AttnParams &p, int pos, int j) {
    return j <= pos && (p.window == 0 || j > (long long)pos - p.window || j < p.sinks);
}

// Whether dimension d of a V row that the row at `pos` sees, and that kv8_clean_v
// may have changed, is NaN: keys of the segment's tiles that one of its rows sees
// and another does not, those of its own positions and of the window's edge.
__device__ __noinline__ bool kv8_patch(const Kv8AttnParams &p, const Kv8Segment &g, int head_dim, int pos, int d) {
    const int last = g.pos0 + g.nodes - 1;
    for (int part = p.window > 0 ? 0 : 1; part < 2; ++part) {
        const int begin = part == 0 ? max(g.low, p.sinks) : g.pos0 + 1;
        const int end = part == 0 ? min(g.pos0, last - p.window) : last;  // the last of them
        for (int j = begin; j <= min(end, g.len - 1); ++j) {
            const int tile = j / kKv8Keys, t = tile < g.sink_tiles ? tile : tile - g.skip;
            if (t < g.t0 || t >= g.t1 || !kv8_sees(p, pos, j)) continue;
            const int page = p.page_table[(long long)g.b * p.max_pages + j / p.page_tokens];
            if (page < 0 || page >= p.num_pages) continue;
            const long long cell = ((long long)page * p.kv_heads + g.kvh) * p.page_tokens + j % p.page_tokens;
            if ((p.v_codes[cell * head_dim + d] & 0x7F) == 0x7F) return true;
        }
    }
    return false;
}

// Joins the parts of the items that shares cut: o = sum_k 2^(m_k - m) o_k / sum_k
// 2^(m_k - m) l_k, in a fixed order. A block per kKv8MergeRows rows of one split
// item; its warps take every eighth part and join through shared memory.
constexpr int kKv8MergeThreads = 256, kKv8MergeRows = 4;

template <int HD, int ROWS>
__global__ void __launch_bounds__(kKv8MergeThreads) kv8_merge_kernel(const Kv8AttnParams p, int ctas) {
    constexpr int kWarps = kKv8MergeThreads / kWarp, V = HD / kWarp;
    static_assert(kKv8MaxCtas <= kKv8MergeThreads, "a thread per listed CTA");
    __shared__ float o_s[kWarps][kKv8MergeRows][HD];
    __shared__ float2 ml_s[kWarps][kKv8MergeRows];
    const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
    pdl_wait();
    pdl_launch_dependents();
    const TreeSplit s = p.splits[blockIdx.x];
    const bool gave_up = (int)threadIdx.x < ctas && p.splits[threadIdx.x].parts < 0;
    if (__syncthreads_or(gave_up)) {
        const long long cells = (long long)min(max(p.row_starts[p.batch], 0), p.rows) * p.q_heads * HD;
        const long long step = (long long)gridDim.x * gridDim.y * kKv8MergeThreads;
        for (long long i = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * kKv8MergeThreads + threadIdx.x; i < cells; i += step) p.out[i] = 0x7FC0u;
        return;
    }
    const int i0 = blockIdx.y * kKv8MergeRows, rows = s.nodes * p.group;
    if (s.parts <= 1 || i0 >= rows) return;
    float m[kKv8MergeRows], l[kKv8MergeRows], o[kKv8MergeRows][V];
#pragma unroll
    for (int i = 0; i < kKv8MergeRows; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.0f;
#pragma unroll
        for (int x = 0; x < V; ++x) o[i][x] = 0.0f;
    }
    auto join = [&](int i, float m2, float l2, const float (&o2)[V]) {
        const float to = fmaxf(m[i], m2);
        const float f = m[i] == -INFINITY ? 0.0f : exp2f(m[i] - to), f2 = m2 == -INFINITY ? 0.0f : exp2f(m2 - to);
        m[i] = to;
        l[i] = l[i] * f + l2 * f2;
#pragma unroll
        for (int x = 0; x < V; ++x) o[i][x] = o[i][x] * f + o2[x] * f2;
    };
#pragma unroll 2
    for (int k = warp; k < s.parts; k += kWarps) {
        const long long slot = k == 0 ? 2 * blockIdx.x + s.first_slot : 2 * (blockIdx.x + k);
        float o2[kKv8MergeRows][V];
        float2 ml[kKv8MergeRows];
#pragma unroll
        for (int i = 0; i < kKv8MergeRows; ++i) {
            const long long row = slot * ROWS + min(i0 + i, rows - 1);
            ml[i] = p.part_ml[row];
#pragma unroll
            for (int x = 0; x < V; ++x) o2[i][x] = p.part_o[row * HD + x * kWarp + lane];
        }
#pragma unroll
        for (int i = 0; i < kKv8MergeRows; ++i) join(i, ml[i].x, ml[i].y, o2[i]);
    }
#pragma unroll
    for (int i = 0; i < kKv8MergeRows; ++i) {
#pragma unroll
        for (int x = 0; x < V; ++x) o_s[warp][i][x * kWarp + lane] = o[i][x];
        if (lane == 0) ml_s[warp][i] = make_float2(m[i], l[i]);
    }
    __syncthreads();
    for (int x = threadIdx.x; x < kKv8MergeRows * HD / 2; x += kKv8MergeThreads) {
        const int i = x / (HD / 2), d = x % (HD / 2) * 2;
        if (i0 + i >= rows) break;
        float top = -INFINITY, sum = 0.0f, a = 0.0f, b = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml_s[w][i].x);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = ml_s[w][i].x == -INFINITY ? 0.0f : exp2f(ml_s[w][i].x - top);
            sum += f * ml_s[w][i].y;
            a += f * o_s[w][i][d];
            b += f * o_s[w][i][d + 1];
        }
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int node = (i0 + i) / p.group, h = (i0 + i) - node * p.group;
        uint32_t w2;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w2) : "f"(b * inv), "f"(a * inv));
        *reinterpret_cast<uint32_t *>(p.out + ((long long)(s.row0 + node) * p.q_heads + s.kvh * p.group + h) * HD + d) = w2;
    }
}

}  // namespace cheetah
