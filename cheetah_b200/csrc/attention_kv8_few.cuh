// Attention over an 8-bit cache for items of few rows (a decoded token, a handful
// of drafted ones): up to R rows, new tokens times the query heads of a KV head.
//
// The keys are the tall side of the products, so few rows cost little:
//   S^T [128 keys x 2R] = K [128 x D] . [q1 | q2]^T         (q's two parts)
//   O^T [D x 3R] += V^T [D x 128 keys] . [w1 | w2 | w3]^T    (the weights')
// K and V are used as they lie in the cache, K with the head's dimensions along
// the products' inner axis, V with the keys along it. A thread has one key of a
// tile and all R rows: its scales are one number each, its exponentials R.
//
// A CTA: warp 0 loads K tiles, warp 1 V tiles and the scales, warp 2 issues the
// MMAs, warp 3 cuts the share into segments and splits q for all but the first;
// then kGroups groups of four warps take turns at the tiles, each with its own O,
// reference m (one per row, agreed on by the group) and sums, joined at a segment's
// end. A group's next S is computed while it works on one, and its next weights are
// written while the last are multiplied. One barrier says that a product is done to
// those who wait for its result and to the loads that wait for its operand's place.
//
// Bound by the loads of K and V where keys are many: 64 sequences of 1000 to 16000
// keys, one row each, 28 + 4 heads of 128, 597 MB: 121 us, 4.9 TB/s. One sequence of
// 700 keys takes 10.9 us: two launches, and a chain of starts, page, tile, S, weights,
// O, join. Three groups instead of two, one barrier per product and faster ends took
// the first case from 151 to 141 us together, loads without divisions to 120 from there;
// rows as the tall side (the other kernel) took 75 us instead of 58 at 32 sequences.
#pragma once

#include "attention_kv8.cuh"

namespace cheetah {

template <int HD, int R>
struct Kv8Few {
    static_assert(R == 8 || R == 16, "more rows are the other kernel's");
    static constexpr int kGroups = 3;
    static constexpr int kThreads = 128 + kGroups * 128;
    static constexpr int kTile = kKv8Keys * HD;                     // one K or V tile
    static constexpr int kAhead = 2;                                // places for a group's weights: one ahead of their product
    // Columns of O^T and rows of the weights: three parts, and what fills them up to a
    // multiple of 16 (nobody reads the columns of those rows, whatever they hold).
    static constexpr int kN = (kKv8Parts * R + 15) / 16 * 16;
    static constexpr int kP = kN * kKv8Keys;                        // the weights of a tile
    static_assert(kP % 1024 == 0, "whole swizzle atoms");
    static constexpr int kPX = kGroups * kAhead * kP;               // at a segment's end the groups' O
    static_assert(kPX >= kGroups * R * HD * 4, "the groups' O");
    static constexpr int kQ = 2 * R * HD;                           // q's parts, one segment's
    // V tiles stay until their weights are there, K tiles only for S: the ring of V
    // is the deeper one.
    static constexpr int kStagesK = (R == 8 ? 6 : 5) * (128 / HD), kStagesV = 6 * (128 / HD);
    // S products ahead of the weights': within the places of S, and such that a
    // barrier's next phase can only end once its group has waited for the last: S of
    // tile x + kStagesK follows the weights of tile x, the products of tile x +
    // kStagesV those of x + kAhead * kGroups, before which the group has waited for x.
    static constexpr int kS = 2 * kGroups < kStagesK ? 2 * kGroups : kStagesK;
    static_assert(kStagesV >= kAhead * kGroups && kStagesK >= kGroups, "phases cannot be lapped");
    static constexpr int kBytes = (kStagesK + kStagesV) * kTile + kPX + 2 * kQ;
    // TMEM: two S per group, so that the next is there when a group has read one, and O.
    static constexpr uint32_t kOCol = kGroups * 4 * R;
    static constexpr uint32_t kCols = kGroups * (4 * R + kN) <= 256 ? 256 : 512;
    static_assert(kGroups * (4 * R + kN) <= (int)kCols, "TMEM columns");
    // Shares of three tiles pay for their join: with six the shortest calls took a fifth more.
    using Cost = Kv8Cost<4, 1, 1, 3>;
    static constexpr int kDims = HD == 128 ? 32 : 16;               // dimensions (lanes) of a warp's part of O^T
};

template <int R, int GROUPS, int STAGES_K, int STAGES_V>
struct Kv8FewShared {
    uint64_t k_full[STAGES_K], s_done[STAGES_K], v_full[STAGES_V], o_done[STAGES_V];
    uint64_t seg_full[kKv8Queue], seg_empty[kKv8Queue], q_full[2], q_empty[2];
    uint64_t p_full[GROUPS][2], vote[GROUPS], exchange, drain;
    Kv8Segment queue[kKv8Queue];
    uint32_t tmem;
    int abort_flag, non_finite;
    uint32_t valid[STAGES_V];              // per V tile: which 16-key blocks hold loaded positions
    alignas(16) float scales[STAGES_V][16];  // K's, then V's
    alignas(16) float q_scale[2][R];
    alignas(16) int far[GROUPS][2][4];               // by place: a warp may be a tile ahead of one that has yet to read
    float top[GROUPS][4][R];               // maxima of a tile whose reference moves
    // A segment's sums have a place of their own: no barrier of a group's warps lies
    // between the last tile's maxima, which all four read, and the first one's sums.
    float sum[GROUPS][4][R];
    float m[GROUPS][R];
};

template <int HD, int R>
constexpr size_t kv8_few_smem() {
    using C = Kv8Few<HD, R>;
    return (size_t)C::kBytes + ((sizeof(Kv8FewShared<R, C::kGroups, C::kStagesK, C::kStagesV>) + 127) & ~size_t(127));
}

// max of a warp's values (NaN ignored).
__device__ __forceinline__ float kv8_warp_max(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

template <int HD, int R>
__global__ void __launch_bounds__(Kv8Few<HD, R>::kThreads, 1)
    attention_kv8_few_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const Kv8AttnParams p) {
    using C = Kv8Few<HD, R>;
    constexpr int kGroups = C::kGroups, kStagesK = C::kStagesK, kStagesV = C::kStagesV;
    constexpr uint32_t kIdescS = umma_idesc_e4m3(kKv8Keys, 2 * R);
    constexpr uint32_t kIdescO = umma_idesc_e4m3(HD, C::kN) | kIdescBE5m2 | (1u << 15);  // V MN-major
    extern __shared__ __align__(1024) uint8_t few_smem[];
    uint8_t *k_ring = few_smem, *v_ring = k_ring + kStagesK * C::kTile;
    uint8_t *px = v_ring + kStagesV * C::kTile;
    uint8_t *q_s = px + C::kPX;
    using Shared = Kv8FewShared<R, kGroups, kStagesK, kStagesV>;
    Shared &sh = *reinterpret_cast<Shared *>(few_smem + C::kBytes);
    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStagesK; ++i) {
            mbar_init(smem_u32(&sh.k_full[i]), 1);
            mbar_init(smem_u32(&sh.s_done[i]), 1);
        }
        for (int i = 0; i < kStagesV; ++i) {
            mbar_init(smem_u32(&sh.v_full[i]), 1);
            mbar_init(smem_u32(&sh.o_done[i]), 1);
        }
        for (int i = 0; i < kKv8Queue; ++i) {
            mbar_init(smem_u32(&sh.seg_full[i]), 1);
            mbar_init(smem_u32(&sh.seg_empty[i]), 3 + kGroups * 4);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&sh.q_full[i]), kGroups * 4);
            mbar_init(smem_u32(&sh.q_empty[i]), kGroups * 4);
        }
        for (int g = 0; g < kGroups; ++g) {
            for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&sh.p_full[g][i]), 4);
            mbar_init(smem_u32(&sh.vote[g]), 4);
        }
        mbar_init(smem_u32(&sh.exchange), kGroups * 4);
        mbar_init(smem_u32(&sh.drain), 1);
        sh.abort_flag = 0;
        sh.non_finite = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(C::kCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    pdl_wait();

    auto wait = [&](uint64_t &bar, uint32_t phase) -> bool { return __all_sync(0xFFFFFFFFu, mbar_wait(smem_u32(&bar), phase)); };
    // The role's next segment, once the scheduler has published it.
    bool ok = true;
    auto next = [&](int seg) -> bool {
        ok = wait(sh.seg_full[seg % kKv8Queue], (seg / kKv8Queue) & 1);
        return ok && sh.queue[seg % kKv8Queue].jobs >= 0;
    };
    auto release = [&](int seg) {
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.seg_empty[seg % kKv8Queue]));
    };
    // Row r of a segment's q, by a warp.
    auto split_row = [&](const Kv8Segment &g, int buf, int r) {
        const int node = r / p.group, h = r - node * p.group;
        const uint16_t *src = node < g.nodes ? p.q + (long long)(g.row0 + node) * p.q_stride + (long long)(g.kvh * p.group + h) * HD : nullptr;
        uint8_t *tile = q_s + buf * C::kQ;
        const float scale = kv8_split_row<HD>(src, tile, r, R + r);
        if (lane == 0) sh.q_scale[buf][r] = scale * p.scale_log2;
    };
    int tile_at = 0;   // tiles of the segments before
    int issued = 0;    // producers: tiles requested
    if (warp == 3) {
        Kv8Walk<typename C::Cost> walk;
        walk.init(p);
        int q_count = 0;  // segments with q
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
            if (g.jobs == 0) continue;
            // q in two parts: rows r and R + r of a K-major tile. The first segment's
            // the groups split, which have nothing else to do yet.
            if (q_count++ == 0) continue;
            const int buf = (q_count - 1) & 1;
            ok = wait(sh.q_empty[buf], (((q_count - 1) >> 1) & 1) ^ 1);
            if (!ok) break;
#pragma unroll 4
            for (int r = 0; r < R; ++r) split_row(g, buf, r);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane < kGroups * 4) mbar_arrive(smem_u32(&sh.q_full[buf]));
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
            ok = is_v ? kv8_load_tiles<HD, kStagesV, true>(p, g, map, sh.v_full, sh.o_done, v_ring, C::kTile, sh.scales, sh.valid, tile_at, issued)
                      : kv8_load_tiles<HD, kStagesK, false>(p, g, map, sh.k_full, sh.s_done, k_ring, C::kTile, nullptr, nullptr, tile_at, issued);
            if (!ok) break;
            tile_at += g.jobs;
            release(seg);
        }
        if (!ok) sh.abort_flag = 1;
    } else if (warp == 2) {
        // The whole warp walks, one elected lane issues.
        const bool leader = elect_one();
        const uint64_t k_desc = umma_smem_desc_e4m3<HD>(smem_u32(k_ring)), v_desc = umma_smem_desc_e4m3<HD>(smem_u32(v_ring));
        const uint64_t p_desc = umma_smem_desc_e4m3<128>(smem_u32(px));
        int q_count = 0, k_buf = 0, v_buf = 0;
        uint32_t k_phase = 0, p_phase = 0;  // of p_full a bit per group and place
        int turns = 0;  // tiles of each group before this segment: its S and weights take two places in turn
        for (int seg = 0; next(seg); ++seg) {
            const int jobs = sh.queue[seg % kKv8Queue].jobs;
            const uint64_t q_desc = umma_smem_desc_e4m3<HD>(smem_u32(q_s + (q_count & 1) * C::kQ));
            int s_at = turns & 1, s_left = jobs;  // the next S's group and place, as 2 * group + place
            auto issue_s = [&]() -> bool {
                if (!wait(sh.k_full[k_buf], k_phase)) return false;
                tc_fence_after();
                --s_left;
                if (leader) {
                    const uint64_t kd = k_desc + (uint32_t)(k_buf * C::kTile >> 4);
#pragma unroll
                    for (int k = 0; k < HD / 32; ++k) umma_e4m3(tmem + s_at * 2 * R, kd + 2 * k, q_desc + 2 * k, kIdescS, k > 0 ? 1u : 0u);
                    umma_commit(smem_u32(&sh.s_done[k_buf]));
                }
                __syncwarp();
                s_at += 2;
                if (s_at >= 2 * kGroups) s_at = (s_at & 1) ^ 1;
                if (++k_buf == kStagesK) {
                    k_buf = 0;
                    k_phase ^= 1;
                }
                return true;
            };
            if (jobs > 0) {
                ok = wait(sh.q_full[q_count & 1], (q_count >> 1) & 1);
                for (int i = 0; ok && i < C::kS && s_left > 0; ++i) ok = issue_s();
                int at = turns & 1;
                for (int i = 0; ok && i < jobs; ++i) {
                    // (V has landed: the group has waited for it. A group may be two
                    // tiles ahead of another: its places have barriers of their own.)
                    ok = wait(sh.p_full[0][at], p_phase >> at & 1);
                    if (!ok) break;
                    p_phase ^= 1u << at;
                    tc_fence_after();
                    if (leader) {
                        const uint64_t vd = v_desc + (uint32_t)(v_buf * C::kTile >> 4);
                        const uint64_t pd = p_desc + (uint32_t)(at * C::kP >> 4);
#pragma unroll
                        for (int k = 0; k < kKv8Keys / 32; ++k)
                            umma_e4m3(tmem + C::kOCol + (at >> 1) * C::kN, vd + (uint32_t)(k * 32 * HD >> 4), pd + 2 * k, kIdescO,
                                      (i >= kGroups || k > 0) ? 1u : 0u);
                        umma_commit(smem_u32(&sh.o_done[v_buf]));
                    }
                    __syncwarp();
                    if (++v_buf == kStagesV) v_buf = 0;
                    at += 2;
                    if (at >= 2 * kGroups) at = (at & 1) ^ 1;
                    if (s_left > 0) ok = issue_s();  // where the group has read its S
                }
                if (!ok) break;
                ++q_count;
                turns += (jobs + kGroups - 1) / kGroups;
            }
            release(seg);
        }
        if (!ok) sh.abort_flag = 1;
    } else {
        const int grp = (warp - 4) / 4, quad = warp % 4;
        const int key = quad * 32 + lane;
        const int tid = threadIdx.x - 128;
        const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
        const uint32_t o_addr = tmem + lane_off + C::kOCol + grp * C::kN;
        // This key's byte in rows 0..7 of the weights (8 rows repeat the swizzle).
        uint32_t p_row[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) p_row[r] = smem_u32(px) + grp * C::kAhead * C::kP + e4m3_tile_offset<128>(r, key >> 4) + (key & 15);
        uint32_t vote_phase = 0, x_phase = 0;
        int turns = 0;  // tiles of each group so far: S and weights take two places in turn
        int q_count = 0;
        bool met = true;  // whether every warp has read the groups' O of the segment before
        for (int seg = 0; next(seg); ++seg) {
            const Kv8Segment &g = sh.queue[seg % kKv8Queue];
            const int jobs = g.jobs, rows = g.nodes * p.group;
            uint16_t *out = p.out + ((long long)g.row0 * p.q_heads + g.kvh * p.group) * HD;
            if (jobs == 0) {
                for (int x = tid; x < rows * (HD / 2); x += kGroups * 128) {
                    const int r = x / (HD / 2), node = r / p.group, h = r - node * p.group;
                    *reinterpret_cast<uint32_t *>(out + ((long long)node * p.q_heads + h) * HD + x % (HD / 2) * 2) = 0u;
                }
                release(seg);
                continue;
            }
            if (q_count == 0) {
                for (int r = grp * 4 + quad; r < R; r += kGroups * 4) split_row(g, 0, r);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.q_full[0]));
            }
            ok = wait(sh.q_full[q_count & 1], (q_count >> 1) & 1);
            if (!ok) break;
            const float *q_scale = sh.q_scale[q_count & 1];
            const int pos0 = g.pos0, last = g.pos0 + g.nodes - 1, len = g.len, nodes = g.nodes;
            const int t0 = g.t0, sink_tiles = g.sink_tiles, skip = g.skip;
            // Tiles of which every row sees every key: those that begin up to
            // whole_end, and, in a window, behind whole_low or among the first positions.
            const int whole_end = min(pos0 + 1, len) - kKv8Keys;
            const int whole_low = p.window > 0 ? (int)max(last - (long long)p.window, -1LL) : -1;
            const int whole_sink = p.window > 0 ? min(p.sinks, INT_MAX) - kKv8Keys : INT_MAX;
            // Weights are 2^arg with arg = t + log2(vs) + sub, sub = kKv8TopLog2 - m, large
            // while nothing has been seen.
            constexpr float kNone = 1e30f;
            float sub[R], l[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                sub[r] = kNone;
                l[r] = 0.0f;
            }
            bool first = true;
            // V tiles (and the phase of their barrier, at bit 8) whose products this
            // group has not waited for: the last two, or -1.
            int older = -1, newer = -1;
            auto wait_o = [&](int &which) -> bool {
                const int w = which;
                which = -1;
                return w < 0 || wait(sh.o_done[w & 0xFF], w >> 8);
            };
            int place = turns & 1, v_buf = (tile_at + grp) % kStagesV, k_buf = (tile_at + grp) % kStagesK;
            uint32_t v_phase = ((tile_at + grp) / kStagesV) & 1, k_phase = ((tile_at + grp) / kStagesK) & 1;
#pragma unroll 1
            for (int i = grp; i < jobs; i += kGroups) {
                const int t = t0 + i, p0 = (t < sink_tiles ? t : t + skip) * kKv8Keys;
                ok = wait(sh.v_full[v_buf], v_phase) && wait(sh.s_done[k_buf], k_phase);
                if (!ok) break;
                tc_fence_after();
                const uint32_t s_addr = tmem + lane_off + (2 * grp + place) * 2 * R;
                const uint32_t valid = sh.valid[v_buf];
                const bool whole = p0 <= whole_end && valid == 0xFFu && (p0 > whole_low || p0 <= whole_sink);
                float ks = sh.scales[v_buf][key >> 4], vs = sh.scales[v_buf][8 + (key >> 4)];
                // The rows that see this key: those of nodes [n0, n1).
                int r0 = 0, r1 = R;
                if (!whole) {
                    const int j = p0 + key;
                    int n0 = 0, n1 = nodes;
                    const bool holds = j < len && (valid >> (key >> 4) & 1);
                    n0 = max(j - pos0, 0);
                    if (p.window > 0 && j >= p.sinks) n1 = (int)min((long long)n1, max(j + (long long)p.window - pos0, 0LL));
                    if (!holds) n1 = 0;
                    if (n0 >= n1) ks = vs = 1.0f;  // scales of a block that no row sees may be anything
                    // A cell that a row of the item does not see.
                    if (!holds || n0 > 0 || n1 < nodes) kv8_clean_v<HD>(v_ring + v_buf * C::kTile + key * HD, holds, &sh.non_finite);
                    r0 = n0 * p.group;
                    r1 = n1 * p.group;
                }
                const float log_vs = kv8_log2(vs);
                __syncwarp();  // the loads from TMEM are the whole warp's
                float arg[R];
                // arg without sub.
                auto scores = [&]() {
                    float s[2 * R];
#pragma unroll
                    for (int x = 0; x < 2 * R; x += 8) tmem_ld8_nowait(s_addr + x, s + x);
                    tmem_wait_ld();
#pragma unroll
                    for (int x = 0; x < R; ++x) {
                        arg[x] = fmaf(s[x] + s[R + x], q_scale[x] * ks, log_vs);
                        if (!whole) arg[x] = x >= r0 && x < r1 ? arg[x] : -INFINITY;
                    }
                };
                scores();
                bool far = false;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    arg[r] += sub[r];
                    far |= arg[r] > kKv8TopLog2 + kKv8RoomLog2;
                }
                far = __any_sync(0xFFFFFFFFu, far);
                if (lane == 0) {
                    *reinterpret_cast<volatile int *>(&sh.far[grp][place][quad]) = far;
                    mbar_arrive(smem_u32(&sh.vote[grp]));
                }
                __syncwarp();
                ok = wait(sh.vote[grp], vote_phase);
                if (!ok) break;
                vote_phase ^= 1;
                const volatile int *votes = sh.far[grp][place];
                if (votes[0] | votes[1] | votes[2] | votes[3]) {
                    // A weight would leave e4m3's range: the rows that have such a
                    // one go over to a whole number above their largest.
                    scores();
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const float top = kv8_warp_max(arg[r]);
                        if (lane == 0) sh.top[grp][quad][r] = top;
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sh.vote[grp]));
                    ok = wait(sh.vote[grp], vote_phase);
                    if (!ok) break;
                    vote_phase ^= 1;
                    // O is this group's once every product into it is done.
                    ok = wait_o(older) && wait_o(newer);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < R; c += 8) {
                        float f[8];
#pragma unroll
                        for (int x = 0; x < 8; ++x) {
                            const int r = c + x;
                            const float top = fmaxf(fmaxf(sh.top[grp][0][r], sh.top[grp][1][r]), fmaxf(sh.top[grp][2][r], sh.top[grp][3][r]));
                            f[x] = 1.0f;
                            if (top + sub[r] > kKv8TopLog2 + kKv8RoomLog2) {
                                const float to = kKv8TopLog2 - ceilf(top);
                                f[x] = sub[r] == kNone ? 0.0f : fast_exp2(to - sub[r]);  // of a whole number: exact
                                sub[r] = to;
                            }
                            l[r] *= f[x];
                            arg[r] += sub[r];
                        }
                        if (!first) {
#pragma unroll
                            for (int part = 0; part < kKv8Parts; ++part) {
                                float o[8];
                                tmem_ld8_nowait(o_addr + part * R + c, o);
                                tmem_wait_ld();
#pragma unroll
                                for (int x = 0; x < 8; ++x) o[x] *= f[x];
                                tmem_st8_nowait(o_addr + part * R + c, o);
                            }
                        }
                    }
                    tmem_wait_st();
                    // (No warp writes `top` again before all four have read it: they
                    // vote first.)
                }
                const float inv_vs = fast_rcp(vs);
                // The weights' place is free once its last product is done, and every
                // warp has read what the segment before left there.
                ok = wait_o(older);
                if (!met) ok = ok && wait(sh.exchange, x_phase);
                if (!ok) break;
                if (!met) x_phase ^= 1;
                met = true;
                const uint32_t p_at = (uint32_t)place * C::kP;
#pragma unroll
                for (int r = 0; r < R; r += 2) {
                    const float w0 = fast_exp2(arg[r]), w1 = fast_exp2(arg[r + 1]);
                    l[r] = fmaf(w0, inv_vs, l[r]);
                    l[r + 1] = fmaf(w1, inv_vs, l[r + 1]);
                    uint32_t w = pack_f16x2(w0, w1);
                    const uint32_t at0 = p_row[r % 8] + p_at + r / 8 * 1024, at1 = p_row[(r + 1) % 8] + p_at + (r + 1) / 8 * 1024;
#pragma unroll
                    for (int part = 0; part < kKv8Parts; ++part) {
                        const uint32_t code = part + 1 < kKv8Parts ? cut_e5m2x2(w) : last_e5m2x2(w);
                        st_shared_u8(at0 + part * R * 128, code >> 8);
                        st_shared_u8(at1 + part * R * 128, code >> 24);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.p_full[grp][place]));
                older = newer;
                newer = v_buf | (int)v_phase << 8;
                first = false;
                place ^= 1;
                v_buf += kGroups;
                if (v_buf >= kStagesV) {
                    v_buf -= kStagesV;
                    v_phase ^= 1;
                }
                k_buf += kGroups;
                if (k_buf >= kStagesK) {
                    k_buf -= kStagesK;
                    k_phase ^= 1;
                }
            }
            if (!ok) break;
            tile_at += jobs;
            turns += (jobs + kGroups - 1) / kGroups;
            // The segment's end: the groups' sums and references, then their O, through
            // shared memory.
            auto arrive = [&]() {
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.exchange));
            };
            auto meet = [&]() -> bool {
                const bool all = wait(sh.exchange, x_phase);
                x_phase ^= 1;
                return all;
            };
            if (!met) ok = meet();  // (a group without a tile of this segment)
            met = true;
            if (!ok) break;
            {
                // Sums over the warp's keys: rows go to lanes, half of them at each step.
                float sum = 0.0f;
#pragma unroll
                for (int c = 0; c < R; c += 8) {
                    float v[8];
#pragma unroll
                    for (int x = 0; x < 8; ++x) v[x] = l[c + x];
#pragma unroll
                    for (int step = 4; step >= 1; step >>= 1) {
                        const bool upper = lane & step;
#pragma unroll
                        for (int x = 0; x < step; ++x) {
                            const float give = upper ? v[x] : v[x + step], keep = upper ? v[x + step] : v[x];
                            v[x] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, step);
                        }
                    }
                    v[0] += __shfl_xor_sync(0xFFFFFFFFu, v[0], 8);
                    v[0] += __shfl_xor_sync(0xFFFFFFFFu, v[0], 16);
                    if (lane / 8 == c / 8) sum = v[0];  // row c + lane % 8
                }
                if (lane < R) sh.sum[grp][quad][lane] = sum;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (lane == r && quad == 0) sh.m[grp][r] = sub[r] == kNone ? -INFINITY : kKv8TopLog2 - sub[r];
                }
            }
            ok = wait_o(older) && wait_o(newer);
            if (!ok) break;
            tc_fence_after();
            arrive();
            ok = meet();
            if (!ok) break;
            // Lane r: row r's largest reference, this group's factor and the sum.
            const int row_of_lane = lane % R;
            float largest = sh.m[0][row_of_lane];
#pragma unroll
            for (int z = 1; z < kGroups; ++z) largest = fmaxf(largest, sh.m[z][row_of_lane]);
            float factor = 0.0f, sum = 0.0f;
#pragma unroll
            for (int z = 0; z < kGroups; ++z) {
                const float mz = sh.m[z][row_of_lane];
                const float f = mz == -INFINITY ? 0.0f : fast_exp2(mz - largest);
                if (z == grp) factor = f;
                sum += f * ((sh.sum[z][0][row_of_lane] + sh.sum[z][1][row_of_lane]) + (sh.sum[z][2][row_of_lane] + sh.sum[z][3][row_of_lane]));
            }
            const int slot = g.slot;
            const bool patch = *reinterpret_cast<volatile int *>(&sh.non_finite) != 0;
            float *exch = reinterpret_cast<float *>(px);  // [group][R][HD]
            const int active = min(jobs, kGroups);
            const int d = quad * C::kDims + lane;
            const float inv_sum = sum == 0.0f ? 0.0f : 1.0f / sum;
            if (grp < active) {
#pragma unroll
                for (int c = 0; c < R; c += 8) {
                    float o[8 * kKv8Parts];
                    __syncwarp();  // lanes part at the stores; the loads from TMEM are the whole warp's
#pragma unroll
                    for (int part = 0; part < kKv8Parts; ++part) tmem_ld8_nowait(o_addr + part * R + c, o + 8 * part);
                    tmem_wait_ld();
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        const float f = __shfl_sync(0xFFFFFFFFu, factor, c + x);
                        if (lane < C::kDims) exch[(grp * R + c + x) * HD + d] = (o[x] + (o[8 + x] + o[16 + x])) * f;
                    }
                }
            }
            arrive();
            ok = meet();
            if (!ok) break;
            for (int x = tid; x < R * HD / 2; x += kGroups * 128) {
                // (A row is one warp's or several.)
                const int r = x / (HD / 2), e = x % (HD / 2) * 2;
                const float inv = __shfl_sync(0xFFFFFFFFu, inv_sum, r), row_sum = __shfl_sync(0xFFFFFFFFu, sum, r),
                            row_top = __shfl_sync(0xFFFFFFFFu, largest, r);
                if (r >= rows) continue;
                float a = 0.0f, b = 0.0f;
#pragma unroll
                for (int z = 0; z < kGroups; ++z) {
                    if (z >= active) break;
                    const float2 v = *reinterpret_cast<const float2 *>(exch + (z * R + r) * HD + e);
                    a += v.x;
                    b += v.y;
                }
                const int node = r / p.group, h = r - node * p.group;
                if (patch) {
                    if (kv8_patch(p, g, HD, pos0 + node, e)) a = NAN;
                    if (kv8_patch(p, g, HD, pos0 + node, e + 1)) b = NAN;
                }
                if (slot >= 0) {
                    const long long row = (2LL * blockIdx.x + slot) * R + r;
                    *reinterpret_cast<float2 *>(p.part_o + row * HD + e) = make_float2(a, b);
                    if (e == 0) p.part_ml[row] = make_float2(row_top, row_sum);
                } else {
                    uint32_t w;
                    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b * inv), "f"(a * inv));
                    *reinterpret_cast<uint32_t *>(out + ((long long)node * p.q_heads + h) * HD + e) = w;
                }
            }
            arrive();
            met = false;  // waited for before the next weights
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.q_empty[q_count & 1]));
            ++q_count;
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
            const int stages = warp == 1 ? kStagesV : kStagesK;
            uint64_t *full = warp == 1 ? sh.v_full : sh.k_full;
            for (int at = max(0, issued - stages); at < issued; ++at) mbar_wait(smem_u32(&full[at % stages]), (at / stages) & 1);
        } else if (warp == 2 && elect_one()) {  // the lane that issued the MMAs
            umma_commit(smem_u32(&sh.drain));
            mbar_wait(smem_u32(&sh.drain), 0);
        }
        if (threadIdx.x == C::kThreads - 1) p.splits[blockIdx.x].parts = -1;  // the merge makes the result NaN
        tc_fence_before();
        __syncthreads();
    }
    if (warp == 2) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kCols));
    }
}

}  // namespace cheetah
