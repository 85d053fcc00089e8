// The 8-bit cache format: e4m3 codes, and one f32 scale for the kKv8Block cells
// of a block and KV head. value = code * scale.
#pragma once

#include <stdint.h>

namespace cheetah {

constexpr int kKv8Block = 16;
constexpr int kKv8LeastLog2 = -64;  // log2 of the smallest scale that an append sets

// Four e4m3 codes of f32 values (nearest, ties to even; NaN stays NaN). Values
// beyond 448 become 448.
__device__ __forceinline__ uint32_t pack_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d) {
    return pack_e4m3x2(a, b) | pack_e4m3x2(c, d) << 16;
}

// Two e4m3 codes (the low half of w) as an f16 pair: exact.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t w) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)w));
    return r;
}
// Two f32 as an f16 pair.
__device__ __forceinline__ uint32_t pack_f16x2(float a, float b) {
    uint32_t w;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
    return w;
}
// An e5m2 is the upper byte of an f16, so a pair of f16 >= 0 comes apart into e5m2 parts
// without conversions: three bits of each are cut off, and what remains is exact.
// The parts' codes are the upper bytes of what is returned, and of what
// last_e5m2x2 rounds (half upwards).
__device__ __forceinline__ uint32_t cut_e5m2x2(uint32_t &w) {
    const uint32_t part = w & 0xFF00FF00u;
    asm("sub.f16x2 %0, %0, %1;" : "+r"(w) : "r"(part));
    return part;
}
__device__ __forceinline__ uint32_t last_e5m2x2(uint32_t w) { return w + 0x00800080u; }
// The codes of four values: the upper bytes of two pairs.
__device__ __forceinline__ uint32_t codes_e5m2x4(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7531); }
__device__ __forceinline__ void unpack_e4m3x2(uint32_t w, float &a, float &b) {
    asm("{\n\t.reg .b16 x, y;\n\tmov.b32 {x, y}, %2;\n\tcvt.f32.f16 %0, x;\n\tcvt.f32.f16 %1, y;\n\t}" : "=f"(a), "=f"(b) : "r"(e4m3x2_to_f16x2(w)));
}
__device__ __forceinline__ void unpack_e4m3x4(uint32_t w, float (&v)[4]) {
    unpack_e4m3x2(w, v[0], v[1]);
    unpack_e4m3x2(w >> 16, v[2], v[3]);
}

// f32 that any narrower format rounds as it would round x: cut off, and the last
// bit set where that left something off (it can then not lie on a tie). A
// non-finite value becomes NaN, which has no code but NaN.
__device__ __forceinline__ float round_to_odd(double x) {
    const float f = __double2float_rz(x);
    const uint32_t bits = __float_as_uint(f);
    if ((bits & 0x7F800000u) == 0x7F800000u) return __uint_as_float(0x7FC00000u);
    return (double)f == x ? f : __uint_as_float(bits | 1u);
}

// a * b cut off, and the last bit set where that left something off.
__device__ __forceinline__ float product_to_odd(float a, float b) {
    const float f = __fmul_rz(a, b);
    return fmaf(a, b, -f) != 0.0f ? __uint_as_float(__float_as_uint(f) | 1u) : f;
}

// Whether these are the bits of a power of two whose inverse is a normal number too.
__device__ __forceinline__ bool kv8_power_of_two(uint32_t bits) { return (bits & 0x7FFFFFu) == 0 && bits >= 0x00800000u && bits <= 0x7E800000u; }

// The smallest power of two, 2^kKv8LeastLog2 at least, whose 448-fold reaches the
// magnitude whose f32 bits these are.
__device__ __forceinline__ float kv8_scale_for(uint32_t top_bits) {
    // 448 = 1.75 * 2^8.
    const int e = (int)(top_bits >> 23) - 127 - 8 + ((top_bits & 0x7FFFFFu) > 0x600000u);
    return __uint_as_float((uint32_t)(max(e, kKv8LeastLog2) + 127) << 23);
}

}  // namespace cheetah
