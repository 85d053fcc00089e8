// Attention over an 8-bit cache for items of many rows (prompt chunks, long
// drafts): rows (new tokens times the query heads of a KV head) fill the 128 rows
// of an MMA, in one or two tiles that share the key tiles.
//
//   S [128 rows x 128 keys] = (q1 + q2) K^T          (q's two parts, from shared memory)
//   O [128 rows x D] += (w1 + w2 + w3) V              (the weights' parts, from TMEM)
//
// The roles of the warps and the order of the MMAs are tree_attention's: warps 0
// and 1 load K and V tiles, warp 2 issues the MMAs, warp 3 cuts the share into
// segments, warps 4-11 are two softmax groups with a row per thread. With two row
// tiles the groups share each key tile, with one they take alternate key tiles and
// join at the end. An item of up to 64 (32) rows fills its tile with two (four)
// copies of them: each copy weighs a half (quarter) of a tile's keys, the others'
// weights being 0 in its rows, and the copies join as the groups do. So the four warps
// of a group always share the softmax; the products cost what they cost anyway.
//
// A block's 16 keys share their scales: the scores' factor is one number per row
// and block, and log2 of V's scale is added to the exponents, so a weight is one
// fused operation and one exponential; the sum l takes a block's weights divided by
// its scale again.
//
// Prompts of 2 x 2000 rows behind up to 6000 keys, 28 + 4 heads of 128: 318 us, 627
// TFLOP/s of the formula's operations, of which the splits do S twice and PV three
// times; 333 us where it runs for long, at the power limit (1.86 GHz). Bound by the
// chain S, softmax, PV of a tile (issue slots 42%, tensor pipe 37%, exponentials 33%).
// With weights in two e4m3 parts, which lose long tails, 300 us. One pass with a running
// maximum took 473 us (weights of a tile done again where the reference moved)
// against 335 us of two at the time. 32 sequences of 1 to 9 rows in a window of
// 4096: 57 us, starts and ends of items half of it. What an item does
// once is written in loops: unrolled it took 60.6 us instead of 56.0 at the time.
#pragma once

#include <type_traits>

#include "attention_kv8.cuh"

namespace cheetah {

constexpr int kManyThreads = 384;
constexpr int kManyRows = 128;
// As kTreeLeanRegs, kTreeSoftmaxRegs: 128 x 64 + 256 x 216 is below 384 x 168.
constexpr int kManyLeanRegs = 64, kManySoftmaxRegs = 216;
static_assert(128 * kManyLeanRegs + 256 * kManySoftmaxRegs <= kManyThreads * 168, "register split");
template <int HD>
struct Kv8Many {
    static constexpr int kTile = kKv8Keys * HD;   // one K or V tile, or one part of a Q tile
    static constexpr int kStages = HD == 128 ? 5 : 11;
    static constexpr int kBytes = 4 * kTile + kStages * 2 * kTile;
    static constexpr uint32_t kOCol = 2 * kKv8Keys;
    // TMEM: S_A | S_B | O_A | O_B; the weights' parts take the columns of the S
    // they came from, those of 64 keys in the columns of these.
    static constexpr uint32_t kHalfCol = 64, kPartCol = 16;
    static_assert(kKv8Parts * kPartCol <= kHalfCol, "the parts of 64 keys");
    // Beginning and end of an item cost what 6 to 8 of its tiles do, and a tile of both
    // row tiles twice one. Lower units (6, 2, 3) took 5% more for prompts.
    using Cost = Kv8Cost<16, 2, 4, 4>;
};

template <int STAGES>
struct Kv8ManyShared {
    uint64_t k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES];
    uint64_t seg_full[kKv8Queue], seg_empty[kKv8Queue];
    uint64_t q_full[2], s_full[2], p_full[2], seg_done, exchange, drain;
    Kv8Segment queue[kKv8Queue];
    uint32_t tmem;
    int abort_flag, non_finite;
    uint32_t valid[STAGES];
    alignas(16) float scales[STAGES][16];
    float2 ml[2][kManyRows];  // at a segment's end; at its beginning .x is q's scale
};

template <int HD>
constexpr size_t kv8_many_smem() {
    return (size_t)Kv8Many<HD>::kBytes + ((sizeof(Kv8ManyShared<Kv8Many<HD>::kStages>) + 127) & ~size_t(127));
}

template <int HD>
__global__ void __launch_bounds__(kManyThreads, 1)
    attention_kv8_many_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const Kv8AttnParams p) {
    using C = Kv8Many<HD>;
    constexpr int kStages = C::kStages;
    constexpr uint32_t kIdescS = umma_idesc_e4m3(kManyRows, kKv8Keys);
    constexpr uint32_t kIdescO = umma_idesc_e4m3(kManyRows, HD) | kIdescAE5m2 | (1u << 16);  // V MN-major
    extern __shared__ __align__(1024) uint8_t many_smem[];
    uint8_t *q_s = many_smem, *ring = many_smem + 4 * C::kTile;  // [tile][part], [stage][K, V]
    Kv8ManyShared<kStages> &sh = *reinterpret_cast<Kv8ManyShared<kStages> *>(many_smem + C::kBytes);
    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(smem_u32(&sh.k_full[i]), 1);
            mbar_init(smem_u32(&sh.k_empty[i]), 1);
            mbar_init(smem_u32(&sh.v_full[i]), 1);
            mbar_init(smem_u32(&sh.v_empty[i]), 1);
        }
        for (int i = 0; i < kKv8Queue; ++i) {
            mbar_init(smem_u32(&sh.seg_full[i]), 1);
            mbar_init(smem_u32(&sh.seg_empty[i]), 3 + 8);
        }
        for (int g = 0; g < 2; ++g) {
            mbar_init(smem_u32(&sh.q_full[g]), 4);
            mbar_init(smem_u32(&sh.s_full[g]), 1);
            mbar_init(smem_u32(&sh.p_full[g]), 4);
        }
        mbar_init(smem_u32(&sh.seg_done), 1);
        mbar_init(smem_u32(&sh.exchange), 8);
        mbar_init(smem_u32(&sh.drain), 1);
        sh.abort_flag = 0;
        sh.non_finite = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512u));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    pdl_wait();

    auto wait = [&](uint64_t &bar, uint32_t phase) -> bool { return __all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&bar), phase)); };
    bool ok = true;
    auto next = [&](int seg) -> bool {
        ok = wait(sh.seg_full[seg % kKv8Queue], (seg / kKv8Queue) & 1);
        return ok && sh.queue[seg % kKv8Queue].jobs >= 0;
    };
    auto release = [&](int seg) {
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.seg_empty[seg % kKv8Queue]));
    };
    int tile_at = 0;  // key tiles of the segments before
    int issued = 0;   // producers: tiles requested
    if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kManyLeanRegs));
    if (warp == 3) {
        Kv8Walk<typename C::Cost> walk;
        walk.init(p);
        for (int seg = 0;; ++seg) {
            const Kv8Segment g = walk.next(p);
            ok = wait(sh.seg_empty[seg % kKv8Queue], ((seg / kKv8Queue) & 1) ^ 1);
            if (!ok) break;
            if (lane == 0) {
                sh.queue[seg % kKv8Queue] = g;
                mbar_arrive(smem_u32(&sh.seg_full[seg % kKv8Queue]));
            }
            __syncwarp();
            if (g.jobs < 0) break;
        }
        if (lane == 0) {
            p.splits[blockIdx.x] = walk.split;
            if (!ok) sh.abort_flag = 1;
        }
    } else if (warp < 2) {
        const bool is_v = warp == 1;
        const CUtensorMap *map = is_v ? &v_map : &k_map;
        for (int seg = 0; next(seg); ++seg) {
            const Kv8Segment &g = sh.queue[seg % kKv8Queue];
            ok = is_v ? kv8_load_tiles<HD, kStages, true>(p, g, map, sh.v_full, sh.v_empty, ring + C::kTile, 2 * C::kTile, sh.scales, sh.valid, tile_at, issued)
                      : kv8_load_tiles<HD, kStages, false>(p, g, map, sh.k_full, sh.k_empty, ring, 2 * C::kTile, nullptr, nullptr, tile_at, issued);
            if (!ok) break;
            tile_at += g.jobs;
            release(seg);
        }
        if (!ok) sh.abort_flag = 1;
    } else if (warp == 2) {
        // The whole warp walks, one elected lane issues.
        const bool leader = elect_one();
        uint32_t q_phase = 0, p_phase[2] = {0, 0};
        const uint64_t q_desc = umma_smem_desc_e4m3<HD>(smem_u32(q_s));
        const uint64_t ring_desc = umma_smem_desc_e4m3<HD>(smem_u32(ring));
        for (int seg = 0; next(seg); ++seg) {
            const int tiles = sh.queue[seg % kKv8Queue].jobs;
            const bool two = sh.queue[seg % kKv8Queue].nodes > p.tile_nodes;
            const int jobs = two ? 2 * tiles : tiles;
            auto issue_s = [&](int i) -> bool {
                const int grp = i & 1, at = tile_at + (two ? i >> 1 : i), buf = at % kStages;
                if ((!two || grp == 0) && !wait(sh.k_full[buf], (at / kStages) & 1)) return false;
                tc_fence_after();
                if (leader) {
                    const uint64_t kd = ring_desc + (uint32_t)(2 * buf * C::kTile >> 4);
                    const uint64_t qd = q_desc + (uint32_t)(2 * grp * C::kTile >> 4);
#pragma unroll
                    for (int part = 0; part < 2; ++part) {
#pragma unroll
                        for (int k = 0; k < HD / 32; ++k)
                            umma_e4m3(tmem + grp * kKv8Keys, qd + (uint32_t)(part * C::kTile >> 4) + 2 * k, kd + 2 * k, kIdescS,
                                      part + k > 0 ? 1u : 0u);
                    }
                    umma_commit(smem_u32(&sh.s_full[grp]));
                    if (!two || grp == 1) umma_commit(smem_u32(&sh.k_empty[buf]));
                }
                __syncwarp();
                return true;
            };
            auto issue_pv = [&](int i) -> bool {
                // (V has landed: the group has waited for it.)
                const int grp = i & 1, at = tile_at + (two ? i >> 1 : i), buf = at % kStages;
                if (!wait(sh.p_full[grp], p_phase[grp])) return false;
                p_phase[grp] ^= 1;
                tc_fence_after();
                if (leader) {
                    const uint64_t vd = ring_desc + (uint32_t)((2 * buf + 1) * C::kTile >> 4);
#pragma unroll
                    for (int part = 0; part < kKv8Parts; ++part) {
#pragma unroll
                        for (int k = 0; k < kKv8Keys / 32; ++k)
                            umma_e4m3_ta(tmem + C::kOCol + grp * HD, tmem + grp * kKv8Keys + (k >> 1) * C::kHalfCol + part * C::kPartCol + (k & 1) * 8,
                                         vd + (uint32_t)(k * 32 * HD >> 4), kIdescO, (i > 1 || part + k > 0) ? 1u : 0u);
                    }
                    if (!two || grp == 1) umma_commit(smem_u32(&sh.v_empty[buf]));
                    if (i == jobs - 1) umma_commit(smem_u32(&sh.seg_done));
                }
                __syncwarp();
                return true;
            };
            if (jobs > 0) {
                ok = wait(sh.q_full[0], q_phase) && wait(sh.q_full[1], q_phase);
                q_phase ^= 1;
                if (ok) ok = issue_s(0) && (jobs < 2 || issue_s(1));
                // S(i + 2) goes into the columns that the weights of i lie in.
                for (int i = 0; ok && i < jobs; ++i) ok = issue_pv(i) && (i + 2 >= jobs || issue_s(i + 2));
                if (!ok) break;
                tile_at += tiles;
            }
            release(seg);
        }
        if (!ok) sh.abort_flag = 1;
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManySoftmaxRegs));
        const int grp = (warp - 4) / 4, quad = warp % 4;
        const int r = quad * 32 + lane;
        const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
        const uint32_t s_addr = tmem + lane_off + grp * kKv8Keys;
        const uint32_t o_addr = tmem + lane_off + C::kOCol + grp * HD;
        uint32_t q_phase = 0, s_phase = 0, done_phase = 0, x_phase = 0;
        // Row of a tile to its node: x / group, exact for x < 256 and group <= 32.
        const uint32_t group_inv = 65536u / p.group + 1u;
        auto node_of = [&](int x) -> int { return (int)(x * group_inv >> 16); };
        for (int seg = 0; next(seg); ++seg) {
            const Kv8Segment &g = sh.queue[seg % kKv8Queue];
            const int tiles = g.jobs;
            const bool two = g.nodes > p.tile_nodes;
            const int jobs = two ? 2 * tiles : tiles;
            const int tile_node = two ? grp * p.tile_nodes : 0;  // first of this group's rows
            // The copies of its rows that the tile holds, one after the other; this
            // thread has row `item_row` and, of every key tile, keys `key_part` * part_rows on.
            const int rows = min(g.nodes, p.tile_nodes) * p.group;
            const int part_rows = rows <= 32 ? 32 : (rows <= 64 ? 64 : kManyRows);
            const int item_row = r & (part_rows - 1), key_part = r / part_rows;
            const int node_of_r = node_of(item_row), head_of_r = item_row - node_of_r * p.group;
            const int node = tile_node + node_of_r;
            const bool live = node_of_r < p.tile_nodes && node < g.nodes;
            uint16_t *out_row = p.out + ((long long)(g.row0 + node) * p.q_heads + g.kvh * p.group + head_of_r) * HD;
            if (jobs == 0) {
                if (live && key_part == 0 && (two || grp == 0)) {
#pragma unroll
                    for (int i = 0; i < HD / 8; ++i) reinterpret_cast<uint4 *>(out_row)[i] = make_uint4(0u, 0u, 0u, 0u);
                }
                release(seg);
                continue;
            }
            // q of this group's rows in two parts: a lane has 16 elements of a row at a
            // time, a warp a quarter of the rows, for all copies; four loads are in flight
            // per lane. (Its tile's last product of the segment before is done.)
            {
                constexpr int kCells = HD / 16, kRowsAt = kWarp / kCells, kLoads = 4;
                uint8_t *tile = q_s + 2 * grp * C::kTile;
                const int c = lane % kCells, first = quad * (part_rows / 4), end = first + part_rows / 4;
                const uint16_t *q = p.q + (long long)(g.row0 + tile_node) * p.q_stride + (long long)g.kvh * p.group * HD + c * 16;
#pragma unroll 1
                for (int y0 = first; y0 < end; y0 += kLoads * kRowsAt) {
                    uint4 raw[kLoads][2];
#pragma unroll
                    for (int i = 0; i < kLoads; ++i) {
                        const int y = y0 + i * kRowsAt + lane / kCells, n = node_of(y), h = y - n * p.group;
                        raw[i][0] = raw[i][1] = make_uint4(0u, 0u, 0u, 0u);
                        if (y < end && n < p.tile_nodes && tile_node + n < g.nodes) {
                            const uint4 *src = reinterpret_cast<const uint4 *>(q + n * p.q_stride + h * HD);
                            raw[i][0] = __ldg(src);
                            raw[i][1] = __ldg(src + 1);
                        }
                    }
#pragma unroll 1
                    for (int y1 = y0; y1 < min(y0 + kLoads * kRowsAt, end); y1 += kRowsAt) {
                        const int y = y1 + lane / kCells;
                        uint4 hi, lo;
                        const float scale = kv8_split_q<HD>(raw[0], hi, lo);
#pragma unroll
                        for (int i = 0; i + 1 < kLoads; ++i) raw[i][0] = raw[i + 1][0], raw[i][1] = raw[i + 1][1];
#pragma unroll 1
                        for (int x = y; x < kManyRows; x += part_rows) {
                            const uint32_t at = e4m3_tile_offset<HD>(x, c);
                            *reinterpret_cast<uint4 *>(tile + at) = hi;
                            *reinterpret_cast<uint4 *>(tile + C::kTile + at) = lo;
                        }
                        if (c == 0) sh.ml[grp][y].x = scale * p.scale_log2;
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.q_full[grp]));
                ok = wait(sh.q_full[grp], q_phase);
                if (!ok) break;
                q_phase ^= 1;
            }
            // (A group without a job does not hold up the segment's end, after which the
            // place is written again.)
            const float q_scale = grp < jobs ? sh.ml[grp][item_row].x : 0.0f;
            const bool warp_live = __any_sync(0xFFFFFFFFu, live);
            // Positions of this row, and of this group's first and last.
            const int pos = g.pos0 + node, first_pos = g.pos0 + tile_node, len = g.len;
            const int last_pos = g.pos0 + min(g.nodes, tile_node + p.tile_nodes) - 1;
            float m_run = -INFINITY, l_run = 0.0f;
            for (int i = grp; i < jobs; i += 2) {
                const int tile = two ? i >> 1 : i, at = tile_at + tile, buf = at % kStages;
                const int p0 = g.key0(g.t0 + tile);
                ok = wait(sh.v_full[buf], (at / kStages) & 1);
                if (!ok) break;
                const uint32_t valid = sh.valid[buf];
                const bool masked = p0 + kKv8Keys - 1 > first_pos || p0 + kKv8Keys > len || valid != 0xFFu ||
                                    (p.window > 0 && p0 <= last_pos - (long long)p.window && p0 + kKv8Keys > p.sinks);
                // What the row sees of the tile, 32 keys to a word.
                uint32_t vis[4] = {0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu, 0xFFFFFFFFu};
                if (masked) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int k0 = p0 + 32 * c;
                        uint32_t bits = kv8_low_bits(min(pos + 1, len) - k0);
                        if (p.window > 0) bits &= ~kv8_low_bits((int)max((long long)pos - p.window + 1 - k0, 0LL)) | kv8_low_bits((int)max(p.sinks - (long long)k0, 0LL));
                        bits &= (valid >> (2 * c) & 1 ? 0x0000FFFFu : 0u) | (valid >> (2 * c + 1) & 1 ? 0xFFFF0000u : 0u);
                        vis[c] = live ? bits : 0u;
                    }
                    // This thread's key: of a cell that some row does not see.
                    const int j = p0 + r;
                    const bool holds = j < len && (valid >> (r >> 4) & 1);
                    if (!holds || j > first_pos || (p.window > 0 && j >= p.sinks && j <= last_pos - (long long)p.window))
                        kv8_clean_v<HD>(ring + (2 * buf + 1) * C::kTile + r * HD, holds, &sh.non_finite);
                }
                // log2 and the inverse of V's scales: lane b % 8 works out those of block b.
                const float vs = sh.scales[buf][8 + (lane & 7)];
                const float my_log = __log2f(vs), my_inv = 1.0f / vs;
                ok = wait(sh.s_full[grp], s_phase);
                if (!ok) break;
                s_phase ^= 1;
                tc_fence_after();
                // Keys [k0, k0 + KEYS) of the tile: their maximum first, then their weights.
                // Scores are read 64 keys at a time; of 128, the first half twice.
                auto weigh = [&](auto keys, const int k0, const uint32_t (&vis)[decltype(keys)::value / 32]) {
                    constexpr int KEYS = decltype(keys)::value, kPieces = KEYS > 64 ? 2 : 1, kPiece = KEYS / kPieces;
                    float s[kPiece];
                    float factor[KEYS / 16], add[KEYS / 16];
                    auto load = [&](int piece) {
#pragma unroll
                        for (int c = 0; c < kPiece / 32; ++c) tmem_ld32_nowait(s_addr + k0 + kPiece * piece + 32 * c, s + 32 * c);
                        tmem_wait_ld();
                        if (masked) {
#pragma unroll
                            for (int k = 0; k < kPiece; ++k) s[k] = (vis[piece * (kPiece / 32) + k / 32] >> (k % 32) & 1) ? s[k] : -INFINITY;
                        }
                    };
#pragma unroll
                    for (int b = 0; b < KEYS / 16; ++b) {
                        factor[b] = q_scale * sh.scales[buf][k0 / 16 + b];
                        add[b] = __shfl_sync(0xFFFFFFFFu, my_log, k0 / 16 + b);
                        // Scales of a block that the row sees nothing of may be anything.
                        if (masked && (vis[b / 2] >> (b % 2 * 16) & 0xFFFFu) == 0) factor[b] = 1.0f, add[b] = 0.0f;
                    }
                    float top = -INFINITY;
#pragma unroll
                    for (int piece = 0; piece < kPieces; ++piece) {
                        load(piece);
#pragma unroll
                        for (int b = 0; b < kPiece / 16; ++b) {
                            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                            for (int k = 0; k < 8; ++k) mx[k & 1] = max3(mx[k & 1], s[16 * b + 2 * k], s[16 * b + 2 * k + 1]);
                            const int all = piece * (kPiece / 16) + b;
                            top = fmaxf(top, fmaf(fmaxf(mx[0], mx[1]), factor[all], add[all]));
                        }
                    }
                    const bool far = top > m_run + kKv8RoomLog2;
                    if (__any_sync(0xFFFFFFFFu, far)) {
                        const float m_new = far ? ceilf(top) : m_run;
                        const float f = far ? exp2f(m_run - m_new) : 1.0f;  // 0 from -inf
                        m_run = m_new;
                        l_run *= f;
                        if (i > 1) {
                            // (S(i) has come after the last product into O.)
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
                    if constexpr (KEYS < kKv8Keys) {
                        // The other copies' keys count nothing here.
                        float zero[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int c = 0; c < kKv8Keys; c += 32) {
                            if (c >= k0 && c < k0 + KEYS) continue;
                            const uint32_t at = s_addr + C::kHalfCol * (c / 64) + c % 64 / 4;
#pragma unroll
                            for (int part = 0; part < kKv8Parts; ++part) tmem_st8_nowait(at + part * C::kPartCol, zero);
                        }
                    }
                    const float base = kKv8TopLog2 - (m_run == -INFINITY ? 0.0f : m_run);
#pragma unroll
                    for (int piece = kPieces - 1; piece >= 0; --piece) {
                        if (piece < kPieces - 1) load(piece);
#pragma unroll
                        for (int c = 0; c < kPiece / 32; ++c) {
                            uint32_t code[kKv8Parts][8];
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const int at16 = 2 * c + h, b = piece * (kPiece / 16) + at16;
                                const unsigned long long f2 = pair_f32(factor[b], factor[b]), a2 = pair_f32(add[b] + base, add[b] + base);
                                unsigned long long sums[2] = {0ull, 0ull};
#pragma unroll
                                for (int x = 0; x < 4; ++x) {
                                    uint32_t w[2];
#pragma unroll
                                    for (int y = 0; y < 2; ++y) {
                                        const int k = 16 * at16 + 4 * x + 2 * y;
                                        float e0, e1;
                                        unpair_f32(fma_pair(pair_f32(s[k], s[k + 1]), f2, a2), e0, e1);
                                        e0 = fast_exp2(e0);
                                        e1 = fast_exp2(e1);
                                        sums[y] = add_pair(sums[y], pair_f32(e0, e1));
                                        w[y] = pack_f16x2(e0, e1);
                                    }
#pragma unroll
                                    for (int part = 0; part + 1 < kKv8Parts; ++part) {
                                        const uint32_t cut = cut_e5m2x2(w[0]);
                                        code[part][4 * h + x] = codes_e5m2x4(cut, cut_e5m2x2(w[1]));
                                    }
                                    code[kKv8Parts - 1][4 * h + x] = codes_e5m2x4(last_e5m2x2(w[0]), last_e5m2x2(w[1]));
                                }
                                float s0, s1;
                                unpair_f32(add_pair(sums[0], sums[1]), s0, s1);
                                const float inv = __shfl_sync(0xFFFFFFFFu, my_inv, k0 / 16 + b);
                                const bool any = !masked || (vis[b / 2] >> (16 * h) & 0xFFFFu) != 0;
                                l_run = any ? fmaf(s0 + s1, inv, l_run) : l_run;
                            }
                            const int key = k0 + kPiece * piece + 32 * c;
                            const uint32_t at = s_addr + C::kHalfCol * (key / 64) + key % 64 / 4;
#pragma unroll
                            for (int part = 0; part < kKv8Parts; ++part) tmem_st8_nowait(at + part * C::kPartCol, reinterpret_cast<const float *>(code[part]));
                        }
                    }
                    tmem_wait_st();
                    tc_fence_before();
                };
                if (warp_live) {
                    if (part_rows == kManyRows) weigh(std::integral_constant<int, 128>{}, 0, vis);
                    else if (part_rows == 64) weigh(std::integral_constant<int, 64>{}, 64 * key_part, {key_part ? vis[2] : vis[0], key_part ? vis[3] : vis[1]});
                    else weigh(std::integral_constant<int, 32>{}, 32 * key_part, {key_part & 2 ? (key_part & 1 ? vis[3] : vis[2]) : (key_part & 1 ? vis[1] : vis[0])});
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.p_full[grp]));
            }
            if (!ok) break;
            tile_at += tiles;
            ok = wait(sh.seg_done, done_phase);
            if (!ok) break;
            done_phase ^= 1;
            tc_fence_after();
            // Weights of this row's accumulators: its own, and the other group's
            // where both hold the same row.
            float w_own = 1.0f, w_other = 0.0f, l = l_run, m = m_run;
            if (!two) {
                sh.ml[grp][r] = make_float2(m_run, l_run);
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.exchange));
                ok = wait(sh.exchange, x_phase);
                if (!ok) break;
                x_phase ^= 1;
                // (Copies of a row are part_rows apart.)
                m = -INFINITY;
#pragma unroll 1
                for (int x = item_row; x < kManyRows; x += part_rows) m = fmaxf(m, fmaxf(sh.ml[0][x].x, sh.ml[1][x].x));
                l = 0.0f;
#pragma unroll 1
                for (int x = item_row; x < 2 * kManyRows; x += part_rows) {
                    const float2 ml = sh.ml[x / kManyRows][x % kManyRows];
                    l += ml.x == -INFINITY ? 0.0f : exp2f(ml.x - m) * ml.y;
                }
                const float m_other = sh.ml[grp ^ 1][r].x;
                w_own = m_run == -INFINITY ? 0.0f : exp2f(m_run - m);
                w_other = m_other == -INFINITY ? 0.0f : exp2f(m_other - m);
            }
            if (warp_live) {
                const bool joined = !two && jobs > 1;
                // Where there was one job, only group A has accumulated.
                const uint32_t own = two || joined ? o_addr : tmem + lane_off + C::kOCol;
                const uint32_t other_addr = tmem + lane_off + C::kOCol + (grp ^ 1) * HD;
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                const int slot = g.slot;
                const long long part_row = (long long)(2 * blockIdx.x + max(slot, 0)) * 256 + (two ? grp * kManyRows : 0) + item_row;
                float4 *part = reinterpret_cast<float4 *>(p.part_o) + (part_row / 256) * (HD / 4) * 256 + part_row % 256;
                const uint32_t live_mask = __ballot_sync(0xFFFFFFFFu, live);
                const bool patch = *reinterpret_cast<volatile int *>(&sh.non_finite) != 0;
                // Two row tiles: every column of the own row. One: group A finishes
                // the first half of the columns, B the second.
                const int d0 = two ? 0 : grp * (HD / 2), d1 = two ? HD : d0 + HD / 2;
                if (part_rows < kManyRows) {
                    // The copies' parts meet in q's place, as [column][row].
                    float *meet = reinterpret_cast<float *>(q_s);
#pragma unroll 1
                    for (int c = d0; c < d1; c += 16) {
                        float ov[16];
                        tmem_ld16(own + c, ov);
                        if (joined) {
                            float ox[16];
                            tmem_ld16(other_addr + c, ox);
#pragma unroll
                            for (int k = 0; k < 16; ++k) ov[k] = ov[k] * w_own + ox[k] * w_other;
                        } else {
                            // (Only group A has accumulated.)
#pragma unroll
                            for (int k = 0; k < 16; ++k) ov[k] *= grp == 0 ? w_own : w_other;
                        }
#pragma unroll
                        for (int k = 0; k < 16; ++k) meet[(c + k) * kManyRows + r] = ov[k];
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sh.exchange));
                    ok = wait(sh.exchange, x_phase);
                    if (!ok) break;
                    x_phase ^= 1;
                    // A thread finishes its row's share of its group's columns, 8 at a time.
                    const int share = HD / 2 * part_rows / kManyRows;
#pragma unroll 1
                    for (int c = d0 + key_part * share; live && c < d0 + (key_part + 1) * share; c += 8) {
                        float v[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) v[k] = 0.0f;
#pragma unroll 1
                        for (int x = item_row; x < kManyRows; x += part_rows) {
#pragma unroll
                            for (int k = 0; k < 8; ++k) v[k] += meet[(c + k) * kManyRows + x];
                        }
                        if (patch) {
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                if (kv8_patch(p, g, HD, pos, c + k)) v[k] = NAN;
                            }
                        }
                        if (slot >= 0) {
                            part[(c / 4) * 256] = make_float4(v[0], v[1], v[2], v[3]);
                            part[(c / 4 + 1) * 256] = make_float4(v[4], v[5], v[6], v[7]);
                        } else {
                            *reinterpret_cast<uint4 *>(out_row + c) =
                                make_uint4(pack_bf16(v[0] * inv, v[1] * inv), pack_bf16(v[2] * inv, v[3] * inv),
                                           pack_bf16(v[4] * inv, v[5] * inv), pack_bf16(v[6] * inv, v[7] * inv));
                        }
                    }
                }
#pragma unroll 1
                for (int c = part_rows < kManyRows ? d1 : d0; c < d1; c += 32) {
                    float ov[32];
                    __syncwarp();  // lanes part below where not all are live; the loads from TMEM are the whole warp's
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
                    if (patch && live) {
#pragma unroll
                        for (int k = 0; k < 32; ++k) {
                            if (kv8_patch(p, g, HD, pos, c + k)) ov[k] = NAN;
                        }
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
                if (live && slot >= 0 && key_part == 0 && (two || grp == 0)) p.part_ml[part_row] = make_float2(m, l);
            }
            tc_fence_before();
            // Neither accumulator may be overwritten before both are read, and
            // neither group may fall a segment behind the other's barriers.
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.exchange));
            ok = wait(sh.exchange, x_phase);
            if (!ok) break;
            x_phase ^= 1;
            release(seg);
        }
        if (!ok) sh.abort_flag = 1;
    }
    tc_fence_before();
    __syncthreads();
    pdl_launch_dependents();
    if (sh.abort_flag) {
        // A wait gave up: let this CTA's copies and MMAs still in flight land
        // before its shared memory and TMEM are released (bounded waits).
        if (warp < 2 && lane == 0) {
            uint64_t *full = warp == 1 ? sh.v_full : sh.k_full;
            for (int at = max(0, issued - kStages); at < issued; ++at) mbar_wait(smem_u32(&full[at % kStages]), (at / kStages) & 1);
        } else if (warp == 2 && elect_one()) {  // the lane that issued the MMAs
            umma_commit(smem_u32(&sh.drain));
            mbar_wait(smem_u32(&sh.drain), 0);
        }
        if (threadIdx.x == kManyThreads - 1) p.splits[blockIdx.x].parts = -1;  // the merge makes the result NaN
        tc_fence_before();
        __syncthreads();
    }
    if (warp == 2) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
    }
}

}  // namespace cheetah
