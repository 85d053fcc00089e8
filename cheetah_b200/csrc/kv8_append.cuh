// q/k norm, rotation and the append of K and V to an 8-bit cache, in one launch:
// the first CTAs take the q heads as qk_norm_rope does, the others the K and V
// heads block by block of the cache.
//
//   y = rotate(x * (1/sqrt(mean(x^2) + eps) * w)),   s = 2^ceil(log2(max|y| / 448)),
//   code = e4m3(y / s)
//
// with one s for the cells of a block (kKv8Block) and head. Bound by memory
// where rows are many and by latency where they are few.
//
// A warp takes the new rows of one (block, head, K or V): up to 16 of them stay
// in registers between the maximum and the codes, so a row is read once. Which
// rows share a block is found from the slots of the 31 rows on either side: the
// first of them leads, its warp takes all. Only a block that holds earlier cells
// is read, and only its scale unless that grows; then the codes ahead of the new
// ones are rounded again.
//
// Codes decide between neighbours 1/8 or 1/16 apart, so a value next to the
// border of two must not be moved over it by a rounding: k is computed in 64 bits,
// reduced to f32 so that no second rounding shows (round_to_odd), and divided by
// a power of two.
#pragma once

#include "common.cuh"
#include "kv8.cuh"
#include "qk_norm_rope.cuh"

namespace cheetah {

struct Kv8AppendParams {
    QkNormRopeParams q;      // the q heads (no KV heads), and what K shares with them
    int kv_heads;
    long long q_blocks;      // CTAs that take q
    int group_rows;          // rows among which a warp looks for blocks to take
    uint8_t *k_codes, *v_codes;
    float *k_scales, *v_scales;
};

constexpr int kKv8Reach = 31;   // rows on either side that may share a block
constexpr int kKv8MaxGroup = 16;

template <typename TIN, int HD>
struct Kv8Cfg {
    static constexpr int kVec = 16 / sizeof(TIN);
    static constexpr int kLanes = HD / 2 / kVec;      // lanes of a row: two chunks each
    static constexpr int kRows = kWarp / kLanes;      // rows a warp takes at a time
    static constexpr int kSteps = kKv8Block / kRows;
};

struct Kv8Members {
    int block[kKv8MaxGroup + 2 * kKv8Reach + 2];  // cache block of each row around; -1: not appended
    int row[kKv8Block], cell[kKv8Block];          // of the block at hand
};

__device__ __forceinline__ void store_codes(uint8_t *dst, const uint32_t (&w)[2]) { *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]); }
__device__ __forceinline__ void store_codes(uint8_t *dst, const uint32_t (&w)[1]) { *reinterpret_cast<uint32_t *>(dst) = w[0]; }

// The `count` rows of one block listed in m, of one K or V head.
template <typename TIN, int HD, bool IS_K>
__device__ __forceinline__ void kv8_append_block(const Kv8AppendParams &p, const Kv8Members &m, int block, int count, int first, int kvh) {
    using C = Kv8Cfg<TIN, HD>;
    constexpr int VEC = C::kVec;
    const int lane = threadIdx.x % kWarp;
    const int c = lane % C::kLanes, sub = lane / C::kLanes;
    const int half = p.q.rotary_dim / 2;
    // As qk_norm_rope_rows: the chunks that are rotated against each other, or
    // the halves of what passes through.
    const bool turned = c * VEC < half;
    const int rest = c * VEC - half;
    const int da = turned ? c * VEC : 2 * half + rest;
    const int db = turned ? half + c * VEC : 2 * half + (HD - 2 * half) / 2 + rest;
    const int head = p.q.q_heads + (IS_K ? 0 : p.kv_heads) + kvh;
    const TIN *base = static_cast<const TIN *>(p.q.qkv) + (long long)head * HD;
    uint4 raw[C::kSteps][2];
#pragma unroll
    for (int s = 0; s < C::kSteps; ++s) {
        const int i = s * C::kRows + sub;
        raw[s][0] = raw[s][1] = make_uint4(0u, 0u, 0u, 0u);
        if (i < count) {
            const TIN *row = base + m.row[i] * p.q.qkv_stride;
            raw[s][0] = __ldcs(reinterpret_cast<const uint4 *>(row + da));
            raw[s][1] = __ldcs(reinterpret_cast<const uint4 *>(row + db));
        }
    }
    const int blocks_per_page = p.q.page_tokens / kKv8Block;
    const int page = block / blocks_per_page, part = block - page * blocks_per_page;
    const long long head_at = (long long)page * p.kv_heads + kvh;
    float *scale_at = (IS_K ? p.k_scales : p.v_scales) + head_at * blocks_per_page + part;
    uint8_t *cells = (IS_K ? p.k_codes : p.v_codes) + (head_at * p.q.page_tokens + part * kKv8Block) * HD;
    const float old = first > 0 ? *scale_at : 0.0f;

    float z[C::kSteps][2 * VEC];
    uint32_t top = 0;
#pragma unroll
    for (int s = 0; s < C::kSteps; ++s) {
        float a[VEC], b[VEC];
        widen_chunk<TIN>(raw[s][0], a);
        widen_chunk<TIN>(raw[s][1], b);
        if (IS_K && s * C::kRows < count) {
            double ya[VEC], yb[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                ya[i] = (double)a[i];
                yb[i] = (double)b[i];
            }
            if (p.q.k_norm != nullptr) {
                double ss = 0.0;
#pragma unroll
                for (int i = 0; i < VEC; ++i) ss = fma(ya[i], ya[i], fma(yb[i], yb[i], ss));
#pragma unroll
                for (int o = C::kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
                const double inv = 1.0 / sqrt(ss * (1.0 / HD) + (double)p.q.eps);
                float wa[VEC], wb[VEC];
                load_floats(p.q.k_norm + da, wa);
                load_floats(p.q.k_norm + db, wb);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    ya[i] *= inv * (double)wa[i];
                    yb[i] *= inv * (double)wb[i];
                }
            }
            const int i = s * C::kRows + sub;
            if (turned && i < count) {
                const long long at = (long long)p.q.positions[m.row[i]] * half + da;
                float cs[VEC], sn[VEC];
                load_floats(p.q.rope_cos + at, cs);
                load_floats(p.q.rope_sin + at, sn);
#pragma unroll
                for (int x = 0; x < VEC; ++x) {
                    const double t = ya[x];
                    ya[x] = t * (double)cs[x] - yb[x] * (double)sn[x];
                    yb[x] = yb[x] * (double)cs[x] + t * (double)sn[x];
                }
            }
#pragma unroll
            for (int x = 0; x < VEC; ++x) {
                a[x] = round_to_odd(ya[x]);
                b[x] = round_to_odd(yb[x]);
            }
        }
#pragma unroll
        for (int x = 0; x < VEC; ++x) {
            z[s][x] = a[x];
            z[s][VEC + x] = b[x];
            const uint32_t ma = __float_as_uint(a[x]) & 0x7FFFFFFFu, mb = __float_as_uint(b[x]) & 0x7FFFFFFFu;
            if (ma < 0x7F800000u) top = max(top, ma);
            if (mb < 0x7F800000u) top = max(top, mb);
        }
    }
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    const float need = kv8_scale_for(top);
    const float scale = old > need && old < INFINITY ? old : need;
    if (first > 0 && scale != old) {
        const double ratio = (double)old / (double)scale;
        uint4 *held = reinterpret_cast<uint4 *>(cells);
        for (int x = lane; x < first * (HD / 16); x += kWarp) {
            const uint4 was = held[x];
            uint32_t w[4] = {was.x, was.y, was.z, was.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float v[4];
                unpack_e4m3x4(w[k], v);
#pragma unroll
                for (int y = 0; y < 4; ++y) v[y] = round_to_odd((double)v[y] * ratio);
                w[k] = pack_e4m3x4(v[0], v[1], v[2], v[3]);
            }
            held[x] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    if (lane == 0 && scale != old) *scale_at = scale;
    // Exact but where a scale that was not set here is no power of two.
    const bool power = (__float_as_uint(scale) & 0x7FFFFFu) == 0;
    const float inv = 1.0f / scale;
#pragma unroll
    for (int s = 0; s < C::kSteps; ++s) {
        const int i = s * C::kRows + sub;
        if (i >= count) continue;
        uint8_t *cell = cells + m.cell[i] * HD;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float v[VEC];
#pragma unroll
            for (int x = 0; x < VEC; ++x) {
                const float y = z[s][h * VEC + x];
                v[x] = power ? y * inv : y / scale;
                if ((__float_as_uint(y) & 0x7F800000u) == 0x7F800000u) v[x] = __uint_as_float(0x7FC00000u);
            }
            uint32_t w[VEC / 4];
#pragma unroll
            for (int k = 0; k < VEC / 4; ++k) w[k] = pack_e4m3x4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
            store_codes(cell + (h ? db : da), w);
        }
    }
}

template <typename TIN, int HD, int U>
__global__ void __launch_bounds__(kQkWarps *kWarp) qk_norm_rope_kv8_kernel(const Kv8AppendParams p) {
    if ((long long)blockIdx.x < p.q_blocks) {
        qk_norm_rope_rows<TIN, TIN, HD, U>(p.q, blockIdx.x);
        return;
    }
    __shared__ Kv8Members members[kQkWarps];
    const int lane = threadIdx.x % kWarp;
    Kv8Members &m = members[threadIdx.x / kWarp];
    const long long unit = ((long long)blockIdx.x - p.q_blocks) * kQkWarps + threadIdx.x / kWarp;
    const int part = (int)(unit % (2 * p.kv_heads));
    const long long first_row = unit / (2 * p.kv_heads) * p.group_rows;
    pdl_wait();
    pdl_launch_dependents();
    if (first_row >= p.q.tokens) return;
    const int r0 = (int)first_row;
    const int group = min(p.group_rows, p.q.tokens - r0);
    const int slots_end = p.q.num_pages * p.q.page_tokens;  // at most 2^31 - 1
    for (int i = lane; i < group + 2 * kKv8Reach; i += kWarp) {
        const long long t = (long long)r0 - kKv8Reach + i;
        int block = -1;
        if (t >= 0 && t < p.q.tokens) {
            const int slot = p.q.slots[t], pos = p.q.positions[t];
            if (slot >= 0 && slot < slots_end && pos >= 0 && pos < p.q.max_positions) block = slot / kKv8Block;
        }
        m.block[i] = block;
    }
    __syncwarp();
    bool leads = false;
    if (lane < group) {
        const int mine = m.block[lane + kKv8Reach];
        bool again = false;
#pragma unroll
        for (int j = 0; j < kKv8Reach; ++j) again |= m.block[lane + j] == mine;
        leads = mine >= 0 && !again;
    }
    for (uint32_t left = __ballot_sync(0xFFFFFFFFu, leads); left; left &= left - 1) {
        const int at = __ffs(left) - 1 + kKv8Reach;
        const int block = m.block[at];
        // The rows of the block and their cells (16 at most: cells are distinct).
        const bool mine = m.block[at + lane] == block;  // at + lane stays within the group's reach
        const uint32_t all = __ballot_sync(0xFFFFFFFFu, mine);
        const int ordinal = __popc(all & ((1u << lane) - 1u));
        int cell = kKv8Block;
        if (mine && ordinal < kKv8Block) {
            const int t = r0 + at - kKv8Reach + lane;
            cell = p.q.slots[t] % kKv8Block;
            m.row[ordinal] = t;
            m.cell[ordinal] = cell;
        }
        const int first = (int)__reduce_min_sync(0xFFFFFFFFu, (uint32_t)cell);
        __syncwarp();
        const int count = min(__popc(all), kKv8Block);
        if (part < p.kv_heads) kv8_append_block<TIN, HD, true>(p, m, block, count, first, part);
        else kv8_append_block<TIN, HD, false>(p, m, block, count, first, part - p.kv_heads);
        __syncwarp();  // before the lists are written again
    }
}

}  // namespace cheetah
