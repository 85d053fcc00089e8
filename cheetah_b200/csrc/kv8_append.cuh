// q/k norm, rotation and the append of K and V to an 8-bit cache, in one launch:
// some CTAs take the q heads, the others the K and V heads
// block by block of the cache.
//
//   y = rotate(x * (1/sqrt(mean(x^2) + eps) * w)),   s = 2^ceil(log2(max|y| / 448)),
//   code = e4m3(y / s)
//
// with one s for the cells of a block (kKv8Block) and head. Bound by memory
// where rows are many and by latency where they are few.
//
// A CTA looks among `group_rows` rows for blocks: the first row that has a block leads
// (which rows share one is found from the slots of the 31 rows on either side). A
// warp holds kRows rows in registers between the maximum and the codes, so a row is
// read once. The rows of short blocks lie side by side in a warp, each warp taking
// other heads; a longer block all four warps take together, head by head. Only a
// block that holds earlier cells is read, and only its scale unless that grows; then
// the codes ahead of the new ones are rounded again.
//
// Codes decide between neighbours 1/8 or 1/16 apart, so a value next to the
// border of two must not be moved over it by a rounding. k is computed in f32 with
// a bound on its error; where the values a bound below and above differ in their
// codes (one in 10^4 does) or in the block's scale, or where f32 would not hold an
// intermediate, the rows at hand are computed again in 64 bits, reduced to f32 so
// that no second rounding shows (round_to_odd). Quotients by a power of two are
// exact. All of k in 64 bits took 243 us for 32768 rows of 28 + 2 * 4 heads of 128.
//
// Measured: 583 MB for 32768 rows of 28 + 2 * 4 heads of 128, bf16, 145 us, 4.0
// TB/s: 16 warps an SM, which their registers allow, leave latencies uncovered (issue
// slots 40%, DRAM 45%); 256 sequences of 1 to 7 rows 15.8 us and one row 3.3 us, chains
// of dependent reads (issue slots 13%).
#pragma once

#include "common.cuh"
#include "kv8.cuh"
#include "pair.cuh"
#include "qk_norm_rope.cuh"

namespace cheetah {

struct Kv8AppendParams {
    QkNormRopeParams q;      // the q heads (no KV heads), and what K shares with them
    int kv_heads;
    uint32_t kv_blocks, every;  // CTAs that append, and of how many one does; the others take q
    int group_rows;          // rows among which a CTA looks for blocks to take
    int parts;               // heads of K and V that it takes of them
    uint8_t *k_codes, *v_codes;
    float *k_scales, *v_scales;
};

constexpr int kKv8Reach = 31;   // rows on either side that may share a block
constexpr int kKv8MaxGroup = 16;

template <typename TIN, int HD>
struct Kv8Cfg {
    static constexpr int kVec = 16 / sizeof(TIN);
    static constexpr int kLanes = HD / 2 / kVec;                  // lanes of a row: two chunks each
    static constexpr int kSide = kWarp / kLanes;                  // rows side by side in a warp
    static constexpr int kSteps = kKv8Block > kSide * kQkWarps ? kKv8Block / (kSide * kQkWarps) : 1;
    static constexpr int kRows = kSide * kSteps;                  // rows of a warp
};

// Of a block: f32 bits of an upper bound of the largest magnitude and of the most
// that a value is off by, and the largest magnitude found in 64 bits where those
// leave the scale open.
struct Kv8Top {
    uint32_t top, off, exact;
};

struct Kv8Members {
    int block[kKv8MaxGroup + 2 * kKv8Reach];   // cache block of each row around; -1: not appended
    int row[kQkWarps][kKv8Block], cell[kQkWarps][kKv8Block];  // of the rows at hand
    int of[kQkWarps][kKv8Block];               // and, of short blocks, which block it is and its first new cell
    Kv8Top top[3][kQkWarps];                   // of the parts that teams of warps take, in turn
};

__device__ __forceinline__ void store_codes(uint8_t *dst, const uint32_t (&w)[2]) { *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]); }
__device__ __forceinline__ void store_codes(uint8_t *dst, const uint32_t (&w)[1]) { *reinterpret_cast<uint32_t *>(dst) = w[0]; }

// Four codes times a power of two.
__device__ __forceinline__ uint32_t kv8_rescale(uint32_t codes, float ratio) {
    float v[4];
    unpack_e4m3x4(codes, v);
    return pack_e4m3x4(v[0] * ratio, v[1] * ratio, v[2] * ratio, v[3] * ratio);
}
// Sixteen codes times old / scale, whatever these are.
__device__ __noinline__ uint4 kv8_rescale_exact(uint4 codes, float old, float scale) {
    const double ratio = (double)old / (double)scale;
    uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll 1
    for (int k = 0; k < 4; ++k) {
        float v[4];
        unpack_e4m3x4(w[k], v);
#pragma unroll
        for (int y = 0; y < 4; ++y) v[y] = round_to_odd((double)v[y] * ratio);
        w[k] = pack_e4m3x4(v[0], v[1], v[2], v[3]);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// VEC elements of a 16-byte chunk as f32 pairs.
template <typename T, int VEC>
__device__ __forceinline__ void widen_pairs(const uint4 &raw, unsigned long long *v) {
    float f[VEC];
    widen_chunk<T>(raw, f);
#pragma unroll
    for (int x = 0; x < VEC / 2; ++x) v[x] = pair_f32(f[2 * x], f[2 * x + 1]);
}

// Mean of the squares of a row, of which each of LANES lanes has N pairs.
template <int HD, int LANES, int N>
__device__ __forceinline__ float kv8_mean_square(const unsigned long long *v) {
    unsigned long long sum = 0ull;
#pragma unroll
    for (int x = 0; x < N; ++x) sum = fma_pair(v[x], v[x], sum);
    float lo, hi;
    unpair_f32(sum, lo, hi);
    lo += hi;
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) lo += __shfl_xor_sync(0xFFFFFFFFu, lo, o);
    return lo * (1.0f / HD);
}

// The rotation of a lane's two chunks at a row's position, the norm's weights
// multiplied into it: (a, b) -> (a wa c - b wb s, b wb c + a wa s). Two elements at a
// time; computed once for all heads of the row.
template <int VEC>
struct Kv8Turn {
    unsigned long long wac[VEC / 2], wbs[VEC / 2], wbc[VEC / 2], was[VEC / 2];  // wbs is negative
    float largest;

    __device__ __forceinline__ void load(const QkNormRopeParams &p, const float *norm, long long at, int da, int db) {
        float c[VEC], s[VEC], wa[VEC], wb[VEC];
#pragma unroll
        for (int x = 0; x < VEC; ++x) {
            c[x] = wa[x] = wb[x] = 1.0f;
            s[x] = 0.0f;
        }
        if (at >= 0) {
            load_floats(p.rope_cos + at, c);
            load_floats(p.rope_sin + at, s);
        }
        if (norm != nullptr) {
            load_floats(norm + da, wa);
            load_floats(norm + db, wb);
        }
        largest = 0.0f;
#pragma unroll
        for (int x = 0; x < VEC; ++x) largest = fmaxf(largest, fmaxf(fabsf(wa[x]), fabsf(wb[x])) * fmaxf(fabsf(c[x]), fabsf(s[x])));
#pragma unroll
        for (int x = 0; x < VEC / 2; ++x) {
            wac[x] = pair_f32(wa[2 * x] * c[2 * x], wa[2 * x + 1] * c[2 * x + 1]);
            wbs[x] = pair_f32(-wb[2 * x] * s[2 * x], -wb[2 * x + 1] * s[2 * x + 1]);
            wbc[x] = pair_f32(wb[2 * x] * c[2 * x], wb[2 * x + 1] * c[2 * x + 1]);
            was[x] = pair_f32(wa[2 * x] * s[2 * x], wa[2 * x + 1] * s[2 * x + 1]);
        }
    }
    __device__ __forceinline__ void apply(unsigned long long *v) const {
#pragma unroll
        for (int x = 0; x < VEC / 2; ++x) {
            const unsigned long long a = v[x], b = v[VEC / 2 + x];
            v[x] = fma_pair(a, wac[x], mul_pair(b, wbs[x]));
            v[VEC / 2 + x] = fma_pair(b, wbc[x], mul_pair(a, was[x]));
        }
    }
};

// The q heads of a row: as qk_norm_rope_rows, with the rotation's numbers and the
// weights multiplied once per row and two elements per operation.
template <typename TIN, int HD, int U>
__device__ __forceinline__ void kv8_q_rows(const QkNormRopeParams &p, uint32_t block) {
    using C = Kv8Cfg<TIN, HD>;
    constexpr int VEC = C::kVec, kLanes = C::kLanes, kHeads = C::kSide, kPairs = VEC / 2;
    const int lane = threadIdx.x % kWarp;
    const int c = lane % kLanes, sub = lane / kLanes;
    const uint32_t unit = block * kQkWarps + threadIdx.x / kWarp;  // (the host keeps it below 2^31)
    const int t = (int)(p.row_units == 1 ? unit : unit / (uint32_t)p.row_units);
    const int step0 = (int)(unit - (uint32_t)t * (uint32_t)p.row_units) * p.steps;
    const int half = p.rotary_dim / 2;
    const bool turned = c * VEC < half;
    const int rest = c * VEC - half;
    const int da = turned ? c * VEC : 2 * half + rest;
    const int db = turned ? half + c * VEC : 2 * half + (HD - 2 * half) / 2 + rest;
    pdl_wait();
    pdl_launch_dependents();
    if (t >= p.tokens) return;
    const TIN *row = static_cast<const TIN *>(p.qkv) + t * p.qkv_stride;
    const int step1 = min((p.q_heads + kHeads - 1) / kHeads, step0 + p.steps);
    uint4 raw[U][2];
    auto load_heads = [&](int s0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int head = (s0 + u) * kHeads + sub;
            raw[u][0] = raw[u][1] = make_uint4(0u, 0u, 0u, 0u);
            if (s0 + u < step1 && head < p.q_heads) {
                raw[u][0] = __ldcs(reinterpret_cast<const uint4 *>(row + (long long)head * HD + da));
                raw[u][1] = __ldcs(reinterpret_cast<const uint4 *>(row + (long long)head * HD + db));
            }
        }
    };
    load_heads(step0);
    const int pos = p.positions[t];
    if (pos < 0 || pos >= p.max_positions) return;
    Kv8Turn<VEC> turn;
    turn.load(p, p.q_norm, turned ? (long long)pos * half + da : -1, da, db);
    for (int s0 = step0; s0 < step1; s0 += U) {
        if (s0 > step0) load_heads(s0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s0 + u >= step1) break;
            const int head = (s0 + u) * kHeads + sub;
            unsigned long long v[2 * kPairs];
            widen_pairs<TIN, VEC>(raw[u][0], v);
            widen_pairs<TIN, VEC>(raw[u][1], v + kPairs);
            float inv = 1.0f;
            if (p.q_norm != nullptr) inv = rsqrtf(kv8_mean_square<HD, kLanes, 2 * kPairs>(v) + p.eps);
            turn.apply(v);
            if (head >= p.q_heads) continue;
            float a[VEC], b[VEC];
#pragma unroll
            for (int x = 0; x < kPairs; ++x) {
                const unsigned long long inv2 = pair_f32(inv, inv);
                unpair_f32(mul_pair(v[x], inv2), a[2 * x], a[2 * x + 1]);
                unpair_f32(mul_pair(v[kPairs + x], inv2), b[2 * x], b[2 * x + 1]);
            }
            const long long at = ((long long)t * p.q_heads + head) * HD;
            store_chunk<TIN, VEC, (U > 1)>(p.q_out, at + da, a);
            store_chunk<TIN, VEC, (U > 1)>(p.q_out, at + db, b);
        }
    }
}

// Quotients by `scale` in 64 bits, rounded to odd, of those elements of the two
// chunks that a lane has of a row whose bit is set (chunk b's from bit VEC on): of k
// (is_k), or of the values as they are. All lanes of a warp call; `at` is the offset
// into the rotary table, or negative.
template <typename TIN, int HD>
__device__ __noinline__ void kv8_exact(const Kv8AppendParams &p, bool is_k, uint4 r0, uint4 r1, int da, int db, long long at, float scale,
                                       uint32_t which, float *out) {
    using C = Kv8Cfg<TIN, HD>;
    constexpr int VEC = C::kVec;
    float wide[2][VEC];
    widen_chunk<TIN>(r0, wide[0]);
    widen_chunk<TIN>(r1, wide[1]);
    const bool normed = is_k && p.q.k_norm != nullptr;
    const uint32_t bits = __float_as_uint(scale);
    const bool power = kv8_power_of_two(bits);
    const double by = (double)__uint_as_float((254u << 23) - bits);  // 1 / scale, where that is a power of two
    double inv = 1.0;
    if (normed) {
        double ss[2] = {0.0, 0.0};
#pragma unroll
        for (int x = 0; x < VEC; ++x) {
            ss[0] = fma((double)wide[0][x], (double)wide[0][x], ss[0]);
            ss[1] = fma((double)wide[1][x], (double)wide[1][x], ss[1]);
        }
        ss[0] += ss[1];
#pragma unroll
        for (int o = C::kLanes / 2; o > 0; o >>= 1) ss[0] += __shfl_xor_sync(0xFFFFFFFFu, ss[0], o);
        inv = 1.0 / sqrt(ss[0] * (1.0 / HD) + (double)p.q.eps);
    }
#pragma unroll 1
    for (; which; which &= which - 1) {
        const int i = __ffs(which) - 1, x = i % VEC;
        const bool second = i >= VEC;
        // This element and the one that it is turned with.
        double a = (double)wide[second][x], b = (double)wide[!second][x];
        if (normed) {
            a *= inv * (double)p.q.k_norm[(second ? db : da) + x];
            b *= inv * (double)p.q.k_norm[(second ? da : db) + x];
        }
        if (is_k && at >= 0) {
            const double cs = (double)p.q.rope_cos[at + x], sn = (double)p.q.rope_sin[at + x];
            a = a * cs + b * (second ? sn : -sn);
        }
        out[i] = round_to_odd(power ? a * by : a / (double)scale);
    }
}

// The `count` rows listed in rows and cells, of every part_step'th of parts [part0,
// part1) (K's heads, then V's), one after the other with the next one's loads under
// way. team > 0: they are one block's, as many warps have kRows each, and every warp
// of the CTA is here (with as many parts: part0 may lie past the end). Else they
// are all rows of one or several blocks (mixed: a row in a warp's side, kSide at
// most); block and first are the lane's.
template <typename TIN, int HD>
__device__ __forceinline__ void kv8_append_rows(const Kv8AppendParams &p, const int *rows, const int *cell_of, Kv8Top (*tops)[kQkWarps], int &turn,
                                                int block, int count, int first, int part0, int part1, int part_step, int team, bool mixed) {
    using C = Kv8Cfg<TIN, HD>;
    constexpr int VEC = C::kVec, kSide = C::kSide, kSteps = C::kSteps;
    const int lane = threadIdx.x % kWarp;
    const bool all = team > 0;
    const int warp = threadIdx.x / kWarp, in_team = all ? warp % team : 0, first_row = in_team * C::kRows;
    // Of a warp whose part lies past the end, only the barriers.
    const int rounds = (part1 - (all ? part0 - warp / team : part0) + part_step - 1) / part_step;
    const int c = lane % C::kLanes, sub = first_row + lane / C::kLanes;
    const int half = p.q.rotary_dim / 2;
    // As qk_norm_rope_rows: the chunks that are rotated against each other, or
    // the halves of what passes through.
    const bool turned = c * VEC < half;
    const int rest = c * VEC - half;
    const int da = turned ? c * VEC : 2 * half + rest;
    const int db = turned ? half + c * VEC : 2 * half + (HD - 2 * half) / 2 + rest;
    // Whether this lane's side has the first listed row of its block.
    bool leader = true;
    if (mixed) {
        const int before = __shfl_up_sync(0xFFFFFFFFu, block, C::kLanes);
        leader = block >= 0 && (lane < C::kLanes || before != block);
    }
    const int blocks_per_page = p.q.page_tokens / kKv8Block;
    const int page = block / blocks_per_page, at_block = block - page * blocks_per_page;
    const TIN *src[kSteps];
    long long rope_at[kSteps];  // -1: not rotated
    int cell[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        const int i = s * kSide + sub;
        src[s] = nullptr;
        rope_at[s] = -1;
        cell[s] = 0;
        if (i < count && part0 < part1) {
            src[s] = static_cast<const TIN *>(p.q.qkv) + rows[i] * p.q.qkv_stride + (long long)p.q.q_heads * HD;
            cell[s] = cell_of[i];
            if (turned && part0 < p.kv_heads) rope_at[s] = (long long)p.q.positions[rows[i]] * half + da;
        }
    }
    auto load = [&](int part, uint4 (&r)[kSteps][2]) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            r[s][0] = r[s][1] = make_uint4(0u, 0u, 0u, 0u);
            if (src[s] != nullptr) {
                r[s][0] = __ldcs(reinterpret_cast<const uint4 *>(src[s] + (long long)part * HD + da));
                r[s][1] = __ldcs(reinterpret_cast<const uint4 *>(src[s] + (long long)part * HD + db));
            }
        }
    };
    auto scale_of = [&](int part) -> float * {
        const bool k = part < p.kv_heads;
        return (k ? p.k_scales : p.v_scales) + ((long long)page * p.kv_heads + (k ? part : part - p.kv_heads)) * blocks_per_page + at_block;
    };
    uint4 raw[kSteps][2], next_raw[kSteps][2];
    load(part0, next_raw);
    const bool holds = first > 0 && (!mixed || src[0] != nullptr);
    float next_old = holds && part0 < part1 ? *scale_of(part0) : 0.0f;
    // k's rotation with the norm's weights in it (Kv8Turn), and the largest of its
    // magnitudes.
    constexpr int kPairs = VEC / 2;
    using Pair = unsigned long long;
    Kv8Turn<VEC> turns[kSteps];
    if (part0 < p.kv_heads) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) turns[s].load(p.q, p.q.k_norm, rope_at[s], da, db);
    }
#pragma unroll 1
    for (int round = 0; round < rounds; ++round) {
        const int part = min(part0 + round * part_step, part1 - 1);
        const bool live = part0 + round * part_step < part1;
        const bool is_k = part < p.kv_heads;
        const float old = next_old;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            raw[s][0] = next_raw[s][0];
            raw[s][1] = next_raw[s][1];
        }
        if (part + part_step < part1) {
            load(part + part_step, next_raw);
            if (holds) next_old = *scale_of(part + part_step);
        }
        // Values over the row's factor (chunk a, then b), and what both of a pair of
        // turned ones are off by in units of kOff: the rotation's largest number of |a|
        // + |b| at most. Squares and sums lose 11 steps of 2^-24 (20 additions, halved
        // by the root), the root 3, weights, rotation and factor 4, the bound itself and
        // what is added to it 4: below 32 of them.
        constexpr float kOff = 0x1p-19f;
        Pair z[kSteps][2 * kPairs], off[kSteps][kPairs];
        float factor[kSteps];
        auto exact = [&](int s, float scale) {  // all lanes of a warp
            float t[2 * VEC];
            kv8_exact<TIN, HD>(p, is_k, raw[s][0], raw[s][1], da, db, rope_at[s], scale, (1u << 2 * VEC) - 1u, t);
#pragma unroll
            for (int x = 0; x < 2 * kPairs; ++x) z[s][x] = pair_f32(t[2 * x], t[2 * x + 1]);
#pragma unroll
            for (int x = 0; x < kPairs; ++x) off[s][x] = 0ull;
            factor[s] = 1.0f;
        };
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            widen_pairs<TIN, VEC>(raw[s][0], z[s]);
            widen_pairs<TIN, VEC>(raw[s][1], z[s] + kPairs);
            factor[s] = 1.0f;
            if (!is_k) continue;
            bool plain = true;
            if (p.q.k_norm != nullptr) {
                const float mean = kv8_mean_square<HD, C::kLanes, 2 * kPairs>(z[s]) + p.q.eps;
                plain = mean > 0x1p-100f && mean < 0x1p100f;  // no square was lost
                factor[s] = rsqrtf(mean);
            }
            float most = 0.0f;
#pragma unroll
            for (int x = 0; x < kPairs; ++x) {
                float a0, a1, b0, b1;
                unpair_f32(z[s][x], a0, a1);
                unpair_f32(z[s][kPairs + x], b0, b1);
                const float o0 = fabsf(a0) + fabsf(b0), o1 = fabsf(a1) + fabsf(b1);
                off[s][x] = pair_f32(o0, o1);
                most = fmaxf(most, fmaxf(o0, o1));
            }
            turns[s].apply(z[s]);
            // (A NaN is no lost value: it stays one. An infinity makes `most` one.)
            most *= turns[s].largest;
            plain = plain && most < 0x1p100f && most * factor[s] < 0x1p100f;
            if (__any_sync(0xFFFFFFFFu, src[s] != nullptr && !plain)) exact(s, 1.0f);
        }
        // The largest of the lanes whose rows are of this lane's block.
        auto among = [&](uint32_t v) -> uint32_t {
            if (!mixed) return __reduce_max_sync(0xFFFFFFFFu, v);
#pragma unroll
            for (int o = 1; o < C::kLanes; o <<= 1) v = max(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
            uint32_t most = v;
#pragma unroll
            for (int o = C::kLanes; o < kWarp; o += C::kLanes) {
                const uint32_t theirs = __shfl_xor_sync(0xFFFFFFFFu, v, o);
                if (__shfl_xor_sync(0xFFFFFFFFu, block, o) == block) most = max(most, theirs);
            }
            return most;
        };
        // f32 bits of the largest finite magnitude.
        auto largest = [&]() -> uint32_t {
            float most = 0.0f;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                float row = 0.0f;
#pragma unroll
                for (int x = 0; x < 2 * kPairs; ++x) {
                    float v0, v1;
                    unpair_f32(z[s][x], v0, v1);
                    row = fmaxf(row, fmaxf(fabsf(v0), fabsf(v1)));
                }
                most = fmaxf(most, row * factor[s]);
            }
            if (__any_sync(0xFFFFFFFFu, most == INFINITY)) {
                most = 0.0f;
#pragma unroll
                for (int s = 0; s < kSteps; ++s) {
#pragma unroll
                    for (int x = 0; x < 2 * kPairs; ++x) {
                        float v[2];
                        unpair_f32(z[s][x], v[0], v[1]);
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            if (fabsf(v[y]) < INFINITY) most = fmaxf(most, fabsf(v[y]) * factor[s]);
                            else v[y] = NAN;  // an infinity has no code
                        }
                        z[s][x] = pair_f32(v[0], v[1]);
                    }
                }
            }
            return among(__float_as_uint(most));
        };
        uint32_t top = largest(), most_off = 0;
        if (is_k) {
            float most = 0.0f;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                float row = 0.0f;
#pragma unroll
                for (int x = 0; x < kPairs; ++x) {
                    float v0, v1;
                    unpair_f32(off[s][x], v0, v1);
                    row = fmaxf(row, fmaxf(v0, v1));
                }
                most = fmaxf(most, row * (turns[s].largest * factor[s]));
            }
            most_off = among(__float_as_uint(most));
        }
        Kv8Top *top_s = &tops[turn % 3][all ? warp / team : 0], *next_top_s = &tops[(turn + 1) % 3][warp];
        turn += all;  // (the same in every warp)
        if (all) {
            if (lane == 0) {
                atomicMax(&top_s->top, top);
                if (is_k) atomicMax(&top_s->off, most_off);
            }
            if (lane == 0) *next_top_s = Kv8Top{0u, 0u, 0u};  // read two rounds ago, written next after this barrier
            __syncthreads();
            top = top_s->top;
            most_off = top_s->off;
        }
        float need = kv8_scale_for(top);
        bool redone = false;
        if (is_k) {
            const float gap = __uint_as_float(most_off) * kOff, at = __uint_as_float(top);
            const bool open = !(gap < INFINITY) || kv8_scale_for(__float_as_uint(at + gap)) != kv8_scale_for(__float_as_uint(fmaxf(at - gap, 0.0f)));
            if (__any_sync(0xFFFFFFFFu, open)) {  // (not mixed: all lanes of the block)
#pragma unroll
                for (int s = 0; s < kSteps; ++s) exact(s, 1.0f);
                top = largest();
                if (all && lane == 0) atomicMax(&top_s->exact, top);
                need = kv8_scale_for(top);
                redone = true;
            }
        }
        // (Every warp is here: another team's block may be open, and parts be of K and V.)
        if (all && __syncthreads_or(redone) && redone) need = kv8_scale_for(top_s->exact);
        const long long head_at = (long long)page * p.kv_heads + (is_k ? part : part - p.kv_heads);
        uint8_t *cells = (is_k ? p.k_codes : p.v_codes) + (head_at * p.q.page_tokens + at_block * kKv8Block) * HD;
        const float scale = old > need && old < INFINITY ? old : need;
        // Who rounds held cells again: the team, the warp, or the block's first row's
        // lanes (a mixed block's rows are neighbours).
        const int held_at = all ? in_team * kWarp + lane : (mixed ? c : lane);
        const int held_step = all ? team * kWarp : (mixed ? C::kLanes : kWarp);
        if (first > 0 && scale != old && leader && live) {
            // The quotient of two powers of two, and a code times it, are exact in f32.
            const bool powers = ((__float_as_uint(old) | __float_as_uint(scale)) & 0x007FFFFFu) == 0 && old > 0.0f;
            const float ratio = old / scale;
            uint4 *held = reinterpret_cast<uint4 *>(cells);
#pragma unroll 1
            for (int x = held_at; x < first * (HD / 16); x += held_step) {
                const uint4 was = held[x];
                held[x] = powers ? make_uint4(kv8_rescale(was.x, ratio), kv8_rescale(was.y, ratio), kv8_rescale(was.z, ratio), kv8_rescale(was.w, ratio))
                                 : kv8_rescale_exact(was, old, scale);
            }
        }
        if ((mixed ? c == 0 && leader : lane == 0 && in_team == 0) && scale != old && live) *scale_of(part) = scale;
        // Products by a power of two are exact; a scale that was not set here may be
        // none, and is divided by in 64 bits.
        const uint32_t scale_bits = __float_as_uint(scale);
        const bool power = kv8_power_of_two(scale_bits);
        const float inv = __uint_as_float((254u << 23) - scale_bits);  // of a power of two: exponents add up to 254
        const Pair minus2 = pair_f32(-1.0f, -1.0f);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            uint32_t w[2 * VEC / 4];
            auto pack = [&](Pair lo, Pair hi) -> uint32_t {
                float v[4];
                unpair_f32(lo, v[0], v[1]);
                unpair_f32(hi, v[2], v[3]);
                return pack_e4m3x4(v[0], v[1], v[2], v[3]);
            };
            uint32_t open = power ? 0u : (1u << 2 * VEC) - 1u;  // elements whose code is not decided yet
            const float by = factor[s] * inv;
            const Pair by2 = pair_f32(by, by);
            if (is_k) {
                const float unit = by * (kOff * turns[s].largest);
                const Pair unit2 = pair_f32(unit, unit);
                Pair e[kPairs];
#pragma unroll
                for (int x = 0; x < kPairs; ++x) e[x] = mul_pair(off[s][x], unit2);
#pragma unroll
                for (int k = 0; k < 2 * VEC / 4; ++k) {
                    const Pair v0 = mul_pair(z[s][2 * k], by2), v1 = mul_pair(z[s][2 * k + 1], by2);
                    const Pair e0 = e[2 * k % kPairs], e1 = e[(2 * k + 1) % kPairs];
                    w[k] = pack(add_pair(v0, e0), add_pair(v1, e1));
                    const uint32_t differ = w[k] ^ pack(fma_pair(e0, minus2, v0), fma_pair(e1, minus2, v1));
                    if (differ) {
#pragma unroll
                        for (int y = 0; y < 4; ++y) open |= (differ >> (8 * y) & 0xFFu ? 1u : 0u) << (4 * k + y);
                    }
                }
            } else {
#pragma unroll
                for (int k = 0; k < 2 * VEC / 4; ++k) w[k] = pack(mul_pair(z[s][2 * k], by2), mul_pair(z[s][2 * k + 1], by2));
            }
            if (__any_sync(0xFFFFFFFFu, open)) {
                float t[2 * VEC];
                uint32_t codes[2 * VEC / 4];
                kv8_exact<TIN, HD>(p, is_k, raw[s][0], raw[s][1], da, db, rope_at[s], scale, open, t);
#pragma unroll
                for (int k = 0; k < 2 * VEC / 4; ++k) codes[k] = w[k];
#pragma unroll 1
                for (; open; open &= open - 1) {
                    const int i = __ffs(open) - 1;
                    reinterpret_cast<uint8_t *>(codes)[i] = (uint8_t)pack_e4m3x2(t[i], t[i]);
                }
#pragma unroll
                for (int k = 0; k < 2 * VEC / 4; ++k) w[k] = codes[k];
            }
            if (src[s] == nullptr || !live) continue;
            uint8_t *dst = cells + cell[s] * HD;
            uint32_t half_w[VEC / 4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int k = 0; k < VEC / 4; ++k) half_w[k] = w[h * (VEC / 4) + k];
                store_codes(dst + (h ? db : da), half_w);
            }
        }
    }
}

template <typename TIN, int HD, int U>
__global__ void __launch_bounds__(kQkWarps *kWarp, 4) qk_norm_rope_kv8_kernel(const Kv8AppendParams p) {
    // The CTAs that append lie among those that take q, one to every `every`: their
    // long chains of dependent steps run beside loads and stores that bound the rest.
    const uint32_t unit = blockIdx.x / p.every;
    if (unit >= p.kv_blocks || unit * p.every != blockIdx.x) {
        kv8_q_rows<TIN, HD, U>(p.q, blockIdx.x - min(unit + (unit * p.every < blockIdx.x), p.kv_blocks));
        return;
    }
    __shared__ Kv8Members m;
    const int lane = threadIdx.x % kWarp, warp = threadIdx.x / kWarp;
    const uint32_t splits = (2 * p.kv_heads + p.parts - 1) / p.parts;  // of a group's parts
    const uint32_t rows_at = splits == 1 ? unit : unit / splits;
    const int part0 = (int)(unit - rows_at * splits) * p.parts, part1 = min(part0 + p.parts, 2 * p.kv_heads);
    const int r0 = (int)rows_at * p.group_rows;
    pdl_wait();
    pdl_launch_dependents();
    const int group = min(p.group_rows, p.q.tokens - r0);
    const int slots_end = p.q.num_pages * p.q.page_tokens;  // at most 2^31 - 1
    static_assert(kKv8MaxGroup + 2 * kKv8Reach <= kQkWarps * kWarp, "a thread per row around");
    if ((int)threadIdx.x < group + 2 * kKv8Reach) {
        const long long t = (long long)r0 - kKv8Reach + threadIdx.x;
        int block = -1;
        if (t >= 0 && t < p.q.tokens) {
            const int slot = p.q.slots[t], pos = p.q.positions[t];
            if (slot >= 0 && slot < slots_end && pos >= 0 && pos < p.q.max_positions) block = slot / kKv8Block;
        }
        m.block[threadIdx.x] = block;
    }
    if (threadIdx.x < 3 * kQkWarps) m.top[threadIdx.x / kQkWarps][threadIdx.x % kQkWarps] = Kv8Top{0u, 0u, 0u};
    __syncthreads();
    bool leads = false;
    if (lane < group) {
        const int mine = m.block[lane + kKv8Reach];
        bool again = false;
#pragma unroll
        for (int j = 0; j < kKv8Reach; ++j) again |= m.block[lane + j] == mine;
        leads = mine >= 0 && !again;
    }
    using C = Kv8Cfg<TIN, HD>;
    int turn = 0;
    int *row_s = m.row[warp], *cell_s = m.cell[warp], *of_s = m.of[warp];
    // The rows of short blocks are gathered side by side in a warp, and each warp
    // takes other heads of them; of a longer block teams of warps do.
    uint32_t left = __ballot_sync(0xFFFFFFFFu, leads);
    while (left) {
        int rows = 0, block = -1, first = 0;
        bool mixed = true;
        while (left) {
            const int at = __ffs(left) - 1 + kKv8Reach;
            block = m.block[at];
            // The rows of the block and their cells (16 at most: cells are distinct).
            const bool mine = m.block[at + lane] == block;  // at + lane stays within the group's reach
            const uint32_t all = __ballot_sync(0xFFFFFFFFu, mine);
            const int count = min(__popc(all), kKv8Block);
            if (rows > 0 && rows + count > C::kSide) break;
            left &= left - 1;
            const int ordinal = rows + __popc(all & ((1u << lane) - 1u));
            int cell = kKv8Block;
            if (mine && ordinal < kKv8Block) {
                const int t = r0 + at - kKv8Reach + lane;
                cell = p.q.slots[t] % kKv8Block;
                row_s[ordinal] = t;
                cell_s[ordinal] = cell;
            }
            first = (int)__reduce_min_sync(0xFFFFFFFFu, (uint32_t)cell);
            if (mine && ordinal < kKv8Block) of_s[ordinal] = at << 8 | first;
            rows += count;
            if (rows >= C::kSide) {
                mixed = rows == C::kSide;
                break;
            }
        }
        __syncwarp();
        int team = 0, from = part0 + warp, step = kQkWarps;
        if (mixed) {
            const int side = lane / C::kLanes;
            block = side < rows ? m.block[of_s[side] >> 8] : -1;
            first = side < rows ? of_s[side] & 0xFF : 0;
        } else if (rows > C::kRows) {
            team = rows > 2 * C::kRows ? kQkWarps : 2;
            from = part0 + warp / team;
            step = kQkWarps / team;
        }
        if (team > 0 || from < part1)
            kv8_append_rows<TIN, HD>(p, row_s, cell_s, m.top, turn, block, rows, first, from, part1, step, team, mixed);
        __syncwarp();  // before the lists are written again
    }
}

}  // namespace cheetah
