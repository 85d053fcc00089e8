// Cells of an 8-bit cache back as bf16 or f32 rows: out = code * scale.
//
// Bound by memory. A thread takes 8 codes of K and of V at a time, several of
// them before the first is used: a 16-byte store of bf16 each, side by side
// along the row. 32768 positions of 4 heads of 128, 101 MB: 18.1 us, 5.6 TB/s; 701
// positions 2.0 us, a launch and two dependent reads.
#pragma once

#include "common.cuh"
#include "kv8.cuh"

namespace cheetah {

constexpr int kKv8ReadThreads = 256;
constexpr int kKv8ReadLoads = 2;   // chunks of K and of V in flight per thread

struct Kv8ReadParams {
    const uint8_t *k_codes, *v_codes;
    const float *k_scales, *v_scales;
    int num_pages, page_tokens;
    const int32_t *slots;
    long long chunks;   // tokens * kv_heads * head_dim / 8
    int kv_heads;
    void *k_out, *v_out;
};

template <typename TOUT>
__device__ __forceinline__ void kv8_store(TOUT *dst, uint2 codes, float scale) {
    float a[4], b[4];
    unpack_e4m3x4(codes.x, a);
    unpack_e4m3x4(codes.y, b);
    // Products by a power of two are exact. Another scale's may not fit f32: rounded
    // there to odd first, they are rounded once.
    if (sizeof(TOUT) == 2 && (__float_as_uint(scale) & 0x7FFFFFu) != 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[i] = product_to_odd(a[i], scale);
            b[i] = product_to_odd(b[i], scale);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[i] *= scale;
            b[i] *= scale;
        }
    }
    if constexpr (sizeof(TOUT) == 2) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(a[2 * i + 1]), "f"(a[2 * i]));
            asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[2 + i]) : "f"(b[2 * i + 1]), "f"(b[2 * i]));
        }
        __stcs(reinterpret_cast<uint4 *>(dst), make_uint4(w[0], w[1], w[2], w[3]));
    } else {
        __stcs(reinterpret_cast<float4 *>(dst), make_float4(a[0], a[1], a[2], a[3]));
        __stcs(reinterpret_cast<float4 *>(dst) + 1, make_float4(b[0], b[1], b[2], b[3]));
    }
}

template <typename TOUT, int HD>
__global__ void __launch_bounds__(kKv8ReadThreads) kv8_read_kernel(const Kv8ReadParams p) {
    constexpr int kChunks = HD / 8;
    pdl_wait();
    pdl_launch_dependents();
    const long long first = (long long)blockIdx.x * kKv8ReadThreads * kKv8ReadLoads + threadIdx.x;
    uint2 k[kKv8ReadLoads], v[kKv8ReadLoads];
    float ks[kKv8ReadLoads], vs[kKv8ReadLoads];
#pragma unroll
    for (int u = 0; u < kKv8ReadLoads; ++u) {
        const long long i = first + u * kKv8ReadThreads;
        k[u] = v[u] = make_uint2(0u, 0u);
        ks[u] = vs[u] = 0.0f;
        if (i >= p.chunks) continue;
        const long long cell = i / kChunks;  // (token, head)
        const int t = (int)(cell / p.kv_heads), h = (int)(cell - (long long)t * p.kv_heads);
        const int slot = p.slots[t];
        const int page = slot / p.page_tokens, at = slot - page * p.page_tokens;
        if (slot < 0 || page >= p.num_pages) continue;
        const long long head = (long long)page * p.kv_heads + h;
        const long long code = (head * p.page_tokens + at) * HD + i % kChunks * 8;
        const long long block = head * (p.page_tokens / kKv8Block) + at / kKv8Block;
        k[u] = __ldcs(reinterpret_cast<const uint2 *>(p.k_codes + code));
        v[u] = __ldcs(reinterpret_cast<const uint2 *>(p.v_codes + code));
        ks[u] = p.k_scales[block];
        vs[u] = p.v_scales[block];
    }
#pragma unroll
    for (int u = 0; u < kKv8ReadLoads; ++u) {
        const long long i = first + u * kKv8ReadThreads;
        if (i >= p.chunks) continue;
        kv8_store(static_cast<TOUT *>(p.k_out) + i * 8, k[u], ks[u]);
        kv8_store(static_cast<TOUT *>(p.v_out) + i * 8, v[u], vs[u]);
    }
}

}  // namespace cheetah
