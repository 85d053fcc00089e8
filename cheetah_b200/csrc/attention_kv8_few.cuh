// Attention over an 8-bit cache for items of few rows (a decoded token, a handful
// of drafted ones): up to R rows, new tokens times the query heads of a KV head.
//
// The keys are the tall side of the products, so few rows cost little:
//   S^T [128 keys x 2R] = K [128 x D] . [q1 | q2]^T         (q's two parts)
//   O^T [D x 2R] += V^T [D x 128 keys] . [w1 | w2]^T         (the weights')
// K and V are used as they lie in the cache, K with the head's dimensions along
// the products' inner axis, V with the keys along it. A thread has one key of a
// tile and all R rows: its scales are one number each, its exponentials R.
//
// A CTA: warp 0 loads K tiles, warp 1 V tiles and the scales, warp 2 issues the
// MMAs, warp 3 cuts the share into segments and splits q; then kGroups groups of
// four warps take turns at the tiles, each with its own S, O, reference m (one per
// row, agreed on by the group) and sums, joined at a segment's end.
#pragma once

#include "attention_kv8.cuh"

namespace cheetah {

template <int HD, int R>
struct Kv8Few {
    static constexpr int kGroups = R == 8 ? 4 : (R == 16 ? 3 : 2);
    static constexpr int kThreads = 128 + kGroups * 128;
    static constexpr int kTile = kKv8Keys * HD;                     // one K or V tile
    static constexpr int kP = 2 * R * kKv8Keys;                     // a group's weights
    static constexpr int kX = kGroups * 8 * HD * 4;                 // 8 rows of every group's O
    static constexpr int kPX = kGroups * kP > kX ? kGroups * kP : kX;
    static constexpr int kQ = 2 * R * HD;                           // q's parts, one segment's
    static constexpr int kStages = HD == 128 ? (R == 32 ? 5 : 6) : (R == 32 ? 11 : 12);
    static constexpr int kBytes = kStages * 2 * kTile + kPX + 2 * kQ;
    static constexpr uint32_t kOCol = kGroups * 2 * R;
    static constexpr uint32_t kCols = kGroups * 4 * R <= 128 ? 128 : 256;
    static_assert(kGroups * 4 * R <= (int)kCols, "TMEM columns");
    using Cost = Kv8Cost<2, 1, 1, 6>;
    static constexpr int kDims = HD == 128 ? 32 : 16;               // dimensions (lanes) of a warp's part of O^T
};

template <int R, int GROUPS, int STAGES>
struct Kv8FewShared {
    uint64_t k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES];
    uint64_t seg_full[kKv8Queue], seg_empty[kKv8Queue], q_full[2], q_empty[2];
    uint64_t s_full[GROUPS], p_full[GROUPS], pv_done[GROUPS], vote[GROUPS], exchange, drain;
    Kv8Segment queue[kKv8Queue];
    uint32_t tmem;
    int abort_flag, non_finite;
    uint32_t valid[STAGES];          // per V tile: which 16-key blocks hold loaded positions
    alignas(16) float scales[STAGES][16];  // K's, then V's
    alignas(16) float q_scale[2][R];
    int far[GROUPS][4];
    float top[GROUPS][4][R];         // maxima, at a segment's end sums
    float m[GROUPS][R];
};

template <int HD, int R>
constexpr size_t kv8_few_smem() {
    using C = Kv8Few<HD, R>;
    return (size_t)C::kBytes + ((sizeof(Kv8FewShared<R, C::kGroups, C::kStages>) + 127) & ~size_t(127));
}

// max of a warp's values (NaN ignored).
__device__ __forceinline__ float kv8_warp_max(float v) {
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

template <int HD, int R>
__global__ void __launch_bounds__(Kv8Few<HD, R>::kThreads, 1)
    attention_kv8_few_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const Kv8AttnParams p) {
    using C = Kv8Few<HD, R>;
    constexpr int kGroups = C::kGroups, kStages = C::kStages;
    constexpr uint32_t kIdescS = umma_idesc_e4m3(kKv8Keys, 2 * R);
    constexpr uint32_t kIdescO = umma_idesc_e4m3(HD, 2 * R) | (1u << 15);  // V MN-major
    extern __shared__ __align__(1024) uint8_t few_smem[];
    uint8_t *ring = few_smem;                        // [stage][K, V]
    uint8_t *px = few_smem + kStages * 2 * C::kTile;
    uint8_t *q_s = px + C::kPX;
    using Shared = Kv8FewShared<R, kGroups, kStages>;
    Shared &sh = *reinterpret_cast<Shared *>(few_smem + C::kBytes);
    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(smem_u32(&sh.k_full[i]), 1);
            mbar_init(smem_u32(&sh.k_empty[i]), 1);
            mbar_init(smem_u32(&sh.v_full[i]), 1 + kWarp);
            mbar_init(smem_u32(&sh.v_empty[i]), 1);
        }
        for (int i = 0; i < kKv8Queue; ++i) {
            mbar_init(smem_u32(&sh.seg_full[i]), 1);
            mbar_init(smem_u32(&sh.seg_empty[i]), 3 + kGroups * 4);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&sh.q_full[i]), kWarp);
            mbar_init(smem_u32(&sh.q_empty[i]), 1 + kGroups * 4);
        }
        for (int g = 0; g < kGroups; ++g) {
            mbar_init(smem_u32(&sh.s_full[g]), 1);
            mbar_init(smem_u32(&sh.p_full[g]), 4);
            mbar_init(smem_u32(&sh.pv_done[g]), 1);
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
            // q in two parts: rows r and R + r of a K-major tile. A lane has 16
            // elements (a cell of each part) of a row at a time.
            const int buf = q_count & 1;
            ok = wait(sh.q_empty[buf], ((q_count >> 1) & 1) ^ 1);
            if (!ok) break;
            ++q_count;
            constexpr int kCells = HD / 16, kRowsAt = kWarp / kCells;
            const int rows = g.nodes * p.group;
            uint8_t *dst = q_s + buf * C::kQ;
#pragma unroll 2
            for (int r0 = 0; r0 < R; r0 += kRowsAt) {
                const int r = r0 + lane / kCells, c = lane % kCells;
                uint4 raw[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
                if (r < rows) {
                    const int node = r / p.group, h = r - node * p.group;
                    const uint4 *src = reinterpret_cast<const uint4 *>(p.q + (long long)(g.row0 + node) * p.q_stride +
                                                                       (long long)(g.kvh * p.group + h) * HD + c * 16);
                    raw[0] = __ldg(src);
                    raw[1] = __ldg(src + 1);
                }
                const float scale = kv8_split_q<HD>(raw, dst, dst, r, R + r, c);
                if (c == 0) sh.q_scale[buf][r] = scale * p.scale_log2;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_arrive(smem_u32(&sh.q_full[buf]));
        }
        if (lane == 0) {
            p.splits[blockIdx.x] = walk.split;
            if (!ok) sh.abort_flag = 1;
        }
    } else if (warp < 2) {
        const bool is_v = warp == 1;
        const CUtensorMap *map = is_v ? &v_map : &k_map;
        uint64_t *full = is_v ? sh.v_full : sh.k_full, *empty = is_v ? sh.v_empty : sh.k_empty;
        for (int seg = 0; next(seg); ++seg) {
            const Kv8Segment &g = sh.queue[seg % kKv8Queue];
            ok = kv8_load_tiles<HD, kStages>(p, g, is_v, map, full, empty, ring, sh.scales, sh.valid, tile_at, issued);
            if (!ok) break;
            tile_at += g.jobs;
            release(seg);
        }
        if (!ok) sh.abort_flag = 1;
    } else if (warp == 2) {
        // The whole warp walks, one elected lane issues.
        const bool leader = elect_one();
        const uint64_t ring_desc = umma_smem_desc_e4m3<HD>(smem_u32(ring));
        const uint64_t p_desc = umma_smem_desc_e4m3<128>(smem_u32(px));
        uint32_t p_phase[kGroups] = {};
        int q_count = 0;
        for (int seg = 0; next(seg); ++seg) {
            const int jobs = sh.queue[seg % kKv8Queue].jobs;
            const uint64_t q_desc = umma_smem_desc_e4m3<HD>(smem_u32(q_s + (q_count & 1) * C::kQ));
            auto issue_s = [&](int i, int grp) -> bool {
                const int at = tile_at + i, buf = at % kStages;
                if (!wait(sh.k_full[buf], (at / kStages) & 1)) return false;
                tc_fence_after();
                if (leader) {
                    const uint64_t kd = ring_desc + (uint32_t)(2 * buf * C::kTile >> 4);
#pragma unroll
                    for (int k = 0; k < HD / 32; ++k) umma_e4m3(tmem + grp * 2 * R, kd + 2 * k, q_desc + 2 * k, kIdescS, k > 0 ? 1u : 0u);
                    umma_commit(smem_u32(&sh.s_full[grp]));
                    umma_commit(smem_u32(&sh.k_empty[buf]));
                    if (i == jobs - 1) umma_commit(smem_u32(&sh.q_empty[q_count & 1]));
                }
                __syncwarp();
                return true;
            };
            if (jobs > 0) {
                ok = wait(sh.q_full[q_count & 1], (q_count >> 1) & 1);
                for (int i = 0; ok && i < min(jobs, kGroups); ++i) ok = issue_s(i, i);
                int grp = 0;
                for (int i = 0; ok && i < jobs; ++i) {
                    const int at = tile_at + i, buf = at % kStages;
                    // (V has landed: the group has waited for it.)
                    ok = wait(sh.p_full[grp], p_phase[grp]);
                    if (!ok) break;
                    p_phase[grp] ^= 1;
                    tc_fence_after();
                    if (leader) {
                        const uint64_t vd = ring_desc + (uint32_t)((2 * buf + 1) * C::kTile >> 4);
                        const uint64_t pd = p_desc + (uint32_t)(grp * C::kP >> 4);
#pragma unroll
                        for (int k = 0; k < kKv8Keys / 32; ++k)
                            umma_e4m3(tmem + C::kOCol + grp * 2 * R, vd + (uint32_t)(k * 32 * HD >> 4), pd + 2 * k, kIdescO,
                                      (i >= kGroups || k > 0) ? 1u : 0u);
                        umma_commit(smem_u32(&sh.pv_done[grp]));
                        umma_commit(smem_u32(&sh.v_empty[buf]));
                    }
                    __syncwarp();
                    if (i + kGroups < jobs) ok = issue_s(i + kGroups, grp);
                    if (++grp == kGroups) grp = 0;
                }
                if (!ok) break;
                ++q_count;
                tile_at += jobs;
            }
            release(seg);
        }
        if (!ok) sh.abort_flag = 1;
    } else {
        const int grp = (warp - 4) / 4, quad = warp % 4;
        const int key = quad * 32 + lane;
        const int tid = threadIdx.x - 128;
        const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
        const uint32_t s_addr = tmem + lane_off + grp * 2 * R;
        const uint32_t o_addr = tmem + lane_off + C::kOCol + grp * 2 * R;
        uint8_t *p_row = px + grp * C::kP + (key & 15);   // this key's byte within a cell
        const int p_cell = key >> 4;
        uint32_t s_phase = 0, pv_phase = 0, vote_phase = 0, x_phase = 0;
        int q_count = 0;
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
            ok = wait(sh.q_full[q_count & 1], (q_count >> 1) & 1);
            if (!ok) break;
            const float *q_scale = sh.q_scale[q_count & 1];
            const int pos0 = g.pos0, last = g.pos0 + g.nodes - 1, len = g.len;
            float m[R], l[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                m[r] = -INFINITY;
                l[r] = 0.0f;
            }
            bool first = true;
            for (int i = grp; i < jobs; i += kGroups) {
                const int at = tile_at + i, buf = at % kStages;
                const int p0 = g.key0(g.t0 + i), j = p0 + key;
                ok = wait(sh.v_full[buf], (at / kStages) & 1) && wait(sh.s_full[grp], s_phase);
                if (!ok) break;
                s_phase ^= 1;
                tc_fence_after();
                float s[2 * R];
#pragma unroll
                for (int c = 0; c < 2 * R; c += 8) tmem_ld8_nowait(s_addr + c, s + c);
                // The rows that see this key: those of nodes [n0, n1).
                const uint32_t valid = sh.valid[buf];
                int n0 = 0, n1 = g.nodes;
                const bool whole = p0 + kKv8Keys - 1 <= pos0 && p0 + kKv8Keys <= len && valid == 0xFFu &&
                                   (p.window == 0 || p0 > last - (long long)p.window || p0 + kKv8Keys <= p.sinks);
                float ks = sh.scales[buf][key >> 4], vs = sh.scales[buf][8 + (key >> 4)];
                if (!whole) {
                    const bool holds = j < len && (valid >> (key >> 4) & 1);
                    n0 = max(j - pos0, 0);
                    if (p.window > 0 && j >= p.sinks) n1 = (int)min((long long)n1, max(j + (long long)p.window - pos0, 0LL));
                    if (!holds) n1 = 0;
                    if (n0 >= n1) ks = vs = 1.0f;
                    // A cell that a row of the item does not see.
                    if (!holds || n0 > 0 || n1 < g.nodes) {
                        uint8_t *tile = ring + (2 * buf + 1) * C::kTile;
                        kv8_clean_v<HD>(tile + key * HD, holds, &sh.non_finite);
                    }
                }
                const int r0 = n0 * p.group, r1 = n1 * p.group;
                // Weights' space and O are the group's once its last product is done.
                if (!first) {
                    ok = wait(sh.pv_done[grp], pv_phase);
                    pv_phase ^= 1;
                }
                tmem_wait_ld();
                if (!ok) break;
                tc_fence_after();
                const float lvs = __log2f(vs);
                bool far = false;
                float t[R];
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    t[r] = (s[r] + s[R + r]) * (q_scale[r] * ks);
                    if (!whole) t[r] = r >= r0 && r < r1 ? t[r] : -INFINITY;
                    if (r >= rows) t[r] = -INFINITY;
                    far |= t[r] + lvs > m[r] + kKv8RoomLog2;
                }
                far = __any_sync(0xFFFFFFFFu, far);
                if (lane == 0) {
                    *reinterpret_cast<volatile int *>(&sh.far[grp][quad]) = far;
                    mbar_arrive(smem_u32(&sh.vote[grp]));
                }
                __syncwarp();
                ok = wait(sh.vote[grp], vote_phase);
                if (!ok) break;
                vote_phase ^= 1;
                const volatile int *votes = sh.far[grp];
                if (votes[0] | votes[1] | votes[2] | votes[3]) {
                    // A weight would leave e4m3's range: the rows that have such a
                    // one go over to a whole number above their largest.
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const float top = kv8_warp_max(t[r] + lvs);
                        if (lane == 0) sh.top[grp][quad][r] = top;
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sh.vote[grp]));
                    ok = wait(sh.vote[grp], vote_phase);
                    if (!ok) break;
                    vote_phase ^= 1;
                    float f[R];
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const float top = fmaxf(fmaxf(sh.top[grp][0][r], sh.top[grp][1][r]), fmaxf(sh.top[grp][2][r], sh.top[grp][3][r]));
                        f[r] = 1.0f;
                        if (top > m[r] + kKv8RoomLog2) {
                            const float to = ceilf(top);
                            f[r] = exp2f(m[r] - to);  // 0 from -inf
                            m[r] = to;
                        }
                        l[r] *= f[r];
                    }
                    if (!first) {
#pragma unroll
                        for (int c = 0; c < 2 * R; c += 8) {
                            float o[8];
                            tmem_ld8_nowait(o_addr + c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int x = 0; x < 8; ++x) o[x] *= f[(c + x) % R];
                            tmem_st8_nowait(o_addr + c, o);
                        }
                        tmem_wait_st();
                    }
                    // (No warp votes again before all four have read `top`: their
                    // weights come first.)
                }
                const float vw = vs * exp2f(kKv8TopLog2);
#pragma unroll
                for (int r = 0; r < R; r += 2) {
                    const float e0 = fast_exp2(t[r] - (m[r] == -INFINITY ? 0.0f : m[r]));
                    const float e1 = fast_exp2(t[r + 1] - (m[r + 1] == -INFINITY ? 0.0f : m[r + 1]));
                    l[r] += e0;
                    l[r + 1] += e1;
                    const float w0 = e0 * vw, w1 = e1 * vw;
                    const uint32_t hi = pack_e4m3x2(w0, w1);
                    float h0, h1;
                    unpack_e4m3x2(hi, h0, h1);
                    const uint32_t lo = pack_e4m3x2(w0 - h0, w1 - h1);
                    p_row[e4m3_tile_offset<128>(r, p_cell)] = (uint8_t)hi;
                    p_row[e4m3_tile_offset<128>(r + 1, p_cell)] = (uint8_t)(hi >> 8);
                    p_row[e4m3_tile_offset<128>(R + r, p_cell)] = (uint8_t)lo;
                    p_row[e4m3_tile_offset<128>(R + r + 1, p_cell)] = (uint8_t)(lo >> 8);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.p_full[grp]));
                first = false;
            }
            if (!ok) break;
            tile_at += jobs;
            // The segment's end: the groups' sums and references, then their O,
            // 8 rows at a time, through shared memory.
            if (!first) {
                ok = wait(sh.pv_done[grp], pv_phase);
                pv_phase ^= 1;
                if (!ok) break;
                tc_fence_after();
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float sum = warp_sum(l[r]);
                if (lane == 0) {
                    sh.top[grp][quad][r] = sum;
                    if (quad == 0) sh.m[grp][r] = m[r];
                }
            }
            auto meet = [&]() -> bool {
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.exchange));
                const bool met = wait(sh.exchange, x_phase);
                x_phase ^= 1;
                return met;
            };
            ok = meet();
            if (!ok) break;
            const int slot = g.slot;
            const bool patch = *reinterpret_cast<volatile int *>(&sh.non_finite) != 0;
            float *exch = reinterpret_cast<float *>(px);  // [group][8][HD]: every product that read the weights is done
            const int active = min(jobs, kGroups);
            const int d = quad * C::kDims + lane;
#pragma unroll 1
            for (int c = 0; c < rows; c += 8) {
                if (grp < active) {
                    float o[16];
                    tmem_ld8_nowait(o_addr + c, o);
                    tmem_ld8_nowait(o_addr + R + c, o + 8);
                    tmem_wait_ld();
                    if (lane < C::kDims) {
#pragma unroll
                        for (int x = 0; x < 8; ++x) {
                            float top = sh.m[0][c + x];
#pragma unroll
                            for (int y = 1; y < kGroups; ++y) top = fmaxf(top, sh.m[y][c + x]);
                            const float mine = sh.m[grp][c + x];
                            const float f = mine == -INFINITY ? 0.0f : exp2f(mine - top);
                            exch[(grp * 8 + x) * HD + d] = (o[x] + o[8 + x]) * f;
                        }
                    }
                }
                ok = meet();
                if (!ok) break;
                for (int x = tid; x < 8 * HD / 2; x += kGroups * 128) {
                    const int y = x / (HD / 2), e = x % (HD / 2) * 2, r = c + y;
                    if (r >= rows) break;
                    float top = sh.m[0][r];
#pragma unroll
                    for (int z = 1; z < kGroups; ++z) top = fmaxf(top, sh.m[z][r]);
                    float sum = 0.0f, a = 0.0f, b = 0.0f;
                    for (int z = 0; z < active; ++z) {
                        const float f = sh.m[z][r] == -INFINITY ? 0.0f : exp2f(sh.m[z][r] - top);
                        sum += f * ((sh.top[z][0][r] + sh.top[z][1][r]) + (sh.top[z][2][r] + sh.top[z][3][r]));
                        const float2 v = *reinterpret_cast<const float2 *>(exch + (z * 8 + y) * HD + e);
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
                        if (e == 0) p.part_ml[row] = make_float2(top, sum);
                    } else {
                        const float inv = sum == 0.0f ? 0.0f : exp2f(-kKv8TopLog2) / sum;
                        uint32_t w;
                        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b * inv), "f"(a * inv));
                        *reinterpret_cast<uint32_t *>(out + ((long long)node * p.q_heads + h) * HD + e) = w;
                    }
                }
                ok = meet();
                if (!ok) break;
            }
            if (!ok) break;
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
            uint64_t *full = warp == 1 ? sh.v_full : sh.k_full;
            for (int at = max(0, issued - kStages); at < issued; ++at) mbar_wait(smem_u32(&full[at % kStages]), (at / kStages) & 1);
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
