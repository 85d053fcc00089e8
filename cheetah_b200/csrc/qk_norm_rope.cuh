// Per-head RMSNorm of q and k, rotation at a given position, append of K and
// V at a given slot, in one pass over the fused projection rows.
//
//   y = x * (1/sqrt(mean(x^2) + eps) * w)        (heads with a norm weight)
//   (a, b) -> (a cos - b sin, b cos + a sin)      (pairs i, i + rotary/2)
//
// Bound by memory: every element is read and written once. A lane holds the
// 16-byte chunk of a head's first half and the chunk of its second half that
// it is rotated with, so the rotation needs no exchange and the norm only a
// sum over the head's HD/2/VEC lanes; a warp takes several heads at a time and
// walks over the heads of one row, whose cos/sin chunk and q weights it keeps
// in registers, with the loads of several head groups issued before the first
// is used. f32 arithmetic, one rounding to the output type. 32768 rows of 28 + 2
// * 4 heads of 128 in bf16 take 110 us (621 MB, 5.6 TB/s, 86% of a copy), 1021
// such rows 6.2 us (3.1 TB/s), one row 1.8 us (latency).
#pragma once

#include "common.cuh"

namespace cheetah {

constexpr int kQkWarps = 4;
// Head groups whose loads a warp issues together when it has many (110 us for
// 32768 rows of 28 + 2 * 4 heads of 128; 3: 115, 4: 116, 9: 132).
constexpr int kQkUnroll = 5;

struct QkNormRopeParams {
    const void *qkv;
    long long qkv_stride;
    const float *q_norm, *k_norm;
    float eps;
    const float *rope_cos, *rope_sin;
    int max_positions, rotary_dim;
    const int32_t *positions, *slots;
    int tokens, q_heads, kv_heads;
    void *q_out, *k_pool, *v_pool;
    int num_pages, page_tokens;
    int steps;      // head groups a warp takes
    int row_units;  // warps per row
};

template <int N>
__device__ __forceinline__ void load_floats(const float *src, float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        const float4 f = __ldg(reinterpret_cast<const float4 *>(src) + i);
        v[4 * i] = f.x;
        v[4 * i + 1] = f.y;
        v[4 * i + 2] = f.z;
        v[4 * i + 3] = f.w;
    }
}

// VEC elements of a 16-byte chunk as f32.
template <typename T, int VEC>
__device__ __forceinline__ void widen_chunk(const uint4 &raw, float (&v)[VEC]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 2) {
            v[2 * i] = bf16_lo(w[i]);
            v[2 * i + 1] = bf16_hi(w[i]);
        } else {
            v[i] = __uint_as_float(w[i]);
        }
    }
}

// STREAM: the chunk is the first to leave L2. A long call's rows are gone before
// the attention reads them; a short call's (1021 rows are under 20 MB) still lie
// there while L2 has room.
template <typename T, int VEC, bool STREAM>
__device__ __forceinline__ void store_chunk(void *base, long long at, const float (&v)[VEC]) {
    if constexpr (sizeof(T) == 2) {
        uint32_t w[VEC / 2];
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
        uint16_t *dst = static_cast<uint16_t *>(base) + at;
        if constexpr (VEC == 8 && STREAM) __stcs(reinterpret_cast<uint4 *>(dst), make_uint4(w[0], w[1], w[2], w[3]));
        else if constexpr (VEC == 8) *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        else *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
    } else {
        float4 *dst = reinterpret_cast<float4 *>(static_cast<float *>(base) + at);
#pragma unroll
        for (int i = 0; i < VEC / 4; ++i) dst[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    }
}

// U: head groups loaded together; 1 where a warp has only one.
template <typename TIN, typename TKV, int HD, int U>
__global__ void __launch_bounds__(kQkWarps *kWarp) qk_norm_rope_rows_kernel(const QkNormRopeParams p) {
    constexpr int VEC = 16 / sizeof(TIN);
    constexpr int kLanes = HD / 2 / VEC;        // lanes of a head
    constexpr int kHeads = kWarp / kLanes;      // heads a warp takes at a time
    const int lane = threadIdx.x % kWarp;
    const int c = lane % kLanes, sub = lane / kLanes;
    const long long unit = (long long)blockIdx.x * kQkWarps + threadIdx.x / kWarp;
    const int t = (int)(unit / p.row_units);
    const int step0 = (int)(unit % p.row_units) * p.steps;
    const int heads = p.q_heads + 2 * p.kv_heads;
    const int half = p.rotary_dim / 2;
    // This lane's two chunks of a head: rotated against each other, or the
    // halves of the part that passes through.
    const bool turned = c * VEC < half;
    const int rest = c * VEC - half;
    const int da = turned ? c * VEC : 2 * half + rest;
    const int db = turned ? half + c * VEC : 2 * half + (HD - 2 * half) / 2 + rest;
    pdl_wait();
    pdl_launch_dependents();
    if (t >= p.tokens) return;
    const TIN *row = static_cast<const TIN *>(p.qkv) + t * p.qkv_stride;
    const int steps = (heads + kHeads - 1) / kHeads;
    const int step1 = min(steps, step0 + p.steps);
    uint4 raw[U][2];
    auto load_heads = [&](int s0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int head = (s0 + u) * kHeads + sub;
            raw[u][0] = raw[u][1] = make_uint4(0u, 0u, 0u, 0u);
            if (s0 + u < step1 && head < heads) {
                raw[u][0] = __ldcs(reinterpret_cast<const uint4 *>(row + (long long)head * HD + da));
                raw[u][1] = __ldcs(reinterpret_cast<const uint4 *>(row + (long long)head * HD + db));
            }
        }
    };
    const int pos = p.positions[t];
    const int slot = p.slots[t];
    // Short rows are asked for together with their position (one row 2.06 ->
    // 1.83 us); longer ones would hold too many registers meanwhile (32768 rows of
    // 36 heads of 128: 134 instead of 110 us).
    constexpr bool kEarly = U <= 3;
    if (kEarly) load_heads(step0);
    float wa[VEC], wb[VEC];
    if (p.q_norm) {
        load_floats(p.q_norm + da, wa);
        load_floats(p.q_norm + db, wb);
    }
    if (pos < 0 || pos >= p.max_positions) return;
    const int page = slot / p.page_tokens;
    const bool cell_ok = slot >= 0 && page < p.num_pages;
    float cs[VEC], sn[VEC];
    if (turned) {
        load_floats(p.rope_cos + (long long)pos * half + da, cs);
        load_floats(p.rope_sin + (long long)pos * half + da, sn);
    }
    for (int s0 = step0; s0 < step1; s0 += U) {
        if (!kEarly || s0 > step0) load_heads(s0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s0 + u >= step1) break;
            const int head = (s0 + u) * kHeads + sub;
            const bool is_q = head < p.q_heads;
            const bool is_k = !is_q && head < p.q_heads + p.kv_heads;
            float a[VEC], b[VEC];
            widen_chunk<TIN>(raw[u][0], a);
            widen_chunk<TIN>(raw[u][1], b);
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) ss = fmaf(a[i], a[i], fmaf(b[i], b[i], ss));
#pragma unroll
            for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
            if (head >= heads) continue;
            if (is_q ? p.q_norm != nullptr : is_k && p.k_norm != nullptr) {
                const float inv = 1.0f / sqrtf(ss * (1.0f / HD) + p.eps);
                if (is_q) {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        a[i] *= inv * wa[i];
                        b[i] *= inv * wb[i];
                    }
                } else {
                    float ka[VEC], kb[VEC];
                    load_floats(p.k_norm + da, ka);
                    load_floats(p.k_norm + db, kb);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        a[i] *= inv * ka[i];
                        b[i] *= inv * kb[i];
                    }
                }
            }
            if ((is_q || is_k) && turned) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float x = a[i];
                    a[i] = x * cs[i] - b[i] * sn[i];
                    b[i] = b[i] * cs[i] + x * sn[i];
                }
            }
            if (is_q) {
                const long long at = ((long long)t * p.q_heads + head) * HD;
                store_chunk<TIN, VEC, (U > 1)>(p.q_out, at + da, a);
                store_chunk<TIN, VEC, (U > 1)>(p.q_out, at + db, b);
            } else if (cell_ok) {
                const int kvh = is_k ? head - p.q_heads : head - p.q_heads - p.kv_heads;
                const long long at = (((long long)page * p.kv_heads + kvh) * p.page_tokens + (slot - page * p.page_tokens)) * HD;
                void *pool = is_k ? p.k_pool : p.v_pool;
                store_chunk<TKV, VEC, (U > 1)>(pool, at + da, a);
                store_chunk<TKV, VEC, (U > 1)>(pool, at + db, b);
            }
        }
    }
}

}  // namespace cheetah
