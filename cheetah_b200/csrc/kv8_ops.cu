// The op entries of a step over an 8-bit cache (include/cheetah_cuda.h): q/k
// norm with rotation and 8-bit append, reading back, attention, and the test of
// drafted tokens. Each checks its arguments, launches on the caller's stream and
// keeps nothing.
#include <cuda.h>
#include <cuda_runtime.h>
#include <math.h>

#include <algorithm>
#include <atomic>
#include <string>
#include <type_traits>

#include "attention_kv8.cuh"
#include "attention_kv8_few.cuh"
#include "attention_kv8_many.cuh"
#include "cheetah_cuda.h"
#include "common.cuh"
#include "kv8_append.cuh"
#include "kv8_read.cuh"
#include "launch.cuh"
#include "verify_drafts.cuh"

using cheetah::launch_ex;

static_assert(cheetah::kKv8Block == CHEETAH_CUDA_KV8_BLOCK, "cells that share a scale");

namespace {

bool aligned(const void *p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

// A pool's slots, and its rows of one head, are numbered in 32 bits.
bool pool_in_range(uint32_t num_pages, uint32_t page_tokens, uint32_t kv_heads) {
    return num_pages > 0 && page_tokens > 0 && page_tokens % CHEETAH_CUDA_KV8_BLOCK == 0 &&
           (uint64_t)num_pages * page_tokens * kv_heads <= 0x7FFFFFFFull;
}

template <typename TIN, int HD>
int launch_append(cheetah::Kv8AppendParams p, cudaStream_t stream) {
    constexpr int kHeads = cheetah::kWarp / (HD / 2 / (16 / (int)sizeof(TIN)));
    int device = 0;
    CH_CUDA_TRY(cudaGetDevice(&device));
    // Warps of the q rows as for qk_norm_rope (verify_ops.cu).
    const int steps = (p.q.q_heads + kHeads - 1) / kHeads;
    p.q.steps = (long long)p.q.tokens * steps >= 48ll * cheetah::sm_count(device) ? steps : 1;
    p.q.row_units = (steps + p.q.steps - 1) / p.q.steps;
    const long long q_blocks = ((long long)p.q.tokens * p.q.row_units + cheetah::kQkWarps - 1) / cheetah::kQkWarps;
    // Rows among which a CTA looks for blocks: sixteen where that gives every SM two
    // CTAs, else four. Their heads are shared by as many CTAs as there is room for
    // beside q's (four on an SM), each with four at least, one for each of its warps.
    const long long sms = cheetah::sm_count(device), parts = 2ll * p.kv_heads;
    p.group_rows = p.q.tokens >= 2 * sms * cheetah::kKv8MaxGroup ? cheetah::kKv8MaxGroup : 4;
    const long long groups = ((long long)p.q.tokens + p.group_rows - 1) / p.group_rows;
    const long long splits = std::max(1ll, std::min((parts + cheetah::kQkWarps - 1) / cheetah::kQkWarps, (4 * sms - q_blocks) / groups));
    p.parts = (int)((parts + splits - 1) / splits);
    const long long kv_blocks = groups * ((parts + p.parts - 1) / p.parts), blocks = q_blocks + kv_blocks;
    // Warps are numbered in 31 bits.
    CH_REQUIRE(blocks <= 0x7FFFFFFFll / cheetah::kQkWarps, "cheetah_cuda_op_qk_norm_rope_kv8: too many rows");
    p.kv_blocks = (uint32_t)kv_blocks;
    p.every = (uint32_t)(blocks / kv_blocks);
    auto kernel = p.q.steps == 1  ? cheetah::qk_norm_rope_kv8_kernel<TIN, HD, 1>
                  : p.q.steps <= 3 ? cheetah::qk_norm_rope_kv8_kernel<TIN, HD, 3>
                                   : cheetah::qk_norm_rope_kv8_kernel<TIN, HD, cheetah::kQkUnroll>;
    CH_CUDA_TRY(launch_ex(kernel, dim3((unsigned)blocks), dim3(cheetah::kQkWarps * cheetah::kWarp), 0, stream,
                          true, p));
    return 0;
}

template <typename TOUT, int HD>
int launch_read(const cheetah::Kv8ReadParams &p, cudaStream_t stream) {
    const long long per_block = cheetah::kKv8ReadThreads * cheetah::kKv8ReadLoads;
    const long long blocks = (p.chunks + per_block - 1) / per_block;
    CH_REQUIRE(blocks <= 0x7FFFFFFFll, "cheetah_cuda_op_kv8_read: too many rows");
    CH_CUDA_TRY(launch_ex(cheetah::kv8_read_kernel<TOUT, HD>, dim3((unsigned)blocks), dim3(cheetah::kKv8ReadThreads), 0, stream, true, p));
    return 0;
}

// 2D map over a pool's codes viewed as [rows][head_dim]: boxes of `box_rows` rows
// of one page, swizzled over a row.
int make_codes_map(CUtensorMap *map, const void *base, uint64_t rows, uint32_t head_dim, uint32_t box_rows) {
    auto encode = cheetah::tensor_map_encoder();
    CH_REQUIRE(encode != nullptr, "CUDA backend: cuTensorMapEncodeTiled is unavailable");
    cuuint64_t dims[2] = {head_dim, rows};
    cuuint64_t strides[1] = {(cuuint64_t)head_dim};
    cuuint32_t box[2] = {head_dim, box_rows};
    cuuint32_t estr[2] = {1u, 1u};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE,
                              head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    CH_REQUIRE(r == CUDA_SUCCESS, "CUDA backend: cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")");
    return 0;
}

int attention_ctas(int device) { return std::min(cheetah::sm_count(device), cheetah::kKv8MaxCtas); }

// Workspace of an attention call of `ctas` CTAs: two parts each, of up to two
// row tiles.
struct AttentionWorkspace {
    size_t splits, ml, o, bytes;
};
AttentionWorkspace attention_workspace(int ctas, uint32_t head_dim) {
    auto up = [](size_t x) { return (x + 255) & ~size_t(255); };
    constexpr int kRows = 2 * cheetah::kManyRows;
    AttentionWorkspace w;
    w.splits = 0;
    w.ml = up(ctas * sizeof(cheetah::TreeSplit));
    w.o = w.ml + up((size_t)ctas * 2 * kRows * sizeof(float2));
    w.bytes = w.o + (size_t)ctas * 2 * kRows * head_dim * sizeof(float);
    return w;
}

template <int HD, int R>
int launch_attention_few(const CUtensorMap &k_map, const CUtensorMap &v_map, cheetah::Kv8AttnParams p, int device, int ctas,
                         cudaStream_t stream) {
    static std::atomic<uint64_t> done{0};
    constexpr size_t smem = cheetah::kv8_few_smem<HD, R>();
    static_assert(smem <= 232448, "shared memory of a CTA");
    p.item_nodes = p.tile_nodes = R / p.group;
    CH_CUDA_TRY(cheetah::allow_smem(cheetah::attention_kv8_few_kernel<HD, R>, smem, device, done));
    CH_CUDA_TRY(launch_ex(cheetah::attention_kv8_few_kernel<HD, R>, dim3(ctas), dim3(cheetah::Kv8Few<HD, R>::kThreads), smem,
                          stream, true, k_map, v_map, p));
    CH_CUDA_TRY(launch_ex(cheetah::kv8_merge_kernel<HD, R>, dim3(ctas, R / cheetah::kKv8MergeRows), dim3(cheetah::kKv8MergeThreads),
                          0, stream, true, p, ctas));
    return 0;
}

template <int HD>
int launch_attention_many(const CUtensorMap &k_map, const CUtensorMap &v_map, cheetah::Kv8AttnParams p, int device, int ctas,
                          cudaStream_t stream) {
    static std::atomic<uint64_t> done{0};
    constexpr size_t smem = cheetah::kv8_many_smem<HD>();
    static_assert(smem <= 232448, "shared memory of a CTA");
    p.tile_nodes = cheetah::kManyRows / p.group;
    p.item_nodes = 2 * p.tile_nodes;
    CH_CUDA_TRY(cheetah::allow_smem(cheetah::attention_kv8_many_kernel<HD>, smem, device, done));
    CH_CUDA_TRY(launch_ex(cheetah::attention_kv8_many_kernel<HD>, dim3(ctas), dim3(cheetah::kManyThreads), smem, stream, true, k_map,
                          v_map, p));
    // Parts lie and are listed as tree attention's.
    cheetah::TreeAttnParams t = {};
    t.row_starts = p.row_starts;
    t.batch = p.batch;
    t.rows = p.rows;
    t.q_heads = p.q_heads;
    t.kv_heads = p.kv_heads;
    t.group = p.group;
    t.tile_nodes = p.tile_nodes;
    t.out = p.out;
    t.splits = p.splits;
    t.part_o = reinterpret_cast<float4 *>(p.part_o);
    t.part_ml = p.part_ml;
    CH_CUDA_TRY(launch_ex(cheetah::tree_merge_kernel<HD>, dim3(ctas * cheetah::kTreeMergeCtas), dim3(cheetah::kTreeMergeThreads), 0,
                          stream, true, t, ctas));
    return 0;
}

}  // namespace

extern "C" {

int cheetah_cuda_op_qk_norm_rope_kv8(const CheetahCudaQkNormRopeKv8 *a, void *stream) {
    CH_REQUIRE(a != nullptr && a->qkv && a->rope_cos && a->rope_sin && a->positions && a->slots && a->q_out &&
                   a->k_codes && a->v_codes && a->k_scales && a->v_scales,
               "cheetah_cuda_op_qk_norm_rope_kv8: null argument");
    CH_REQUIRE(a->dtype == CHEETAH_CUDA_KV_BF16 || a->dtype == CHEETAH_CUDA_KV_F32,
               "cheetah_cuda_op_qk_norm_rope_kv8: unknown dtype");
    CH_REQUIRE(a->head_dim == 64 || a->head_dim == 128, "cheetah_cuda_op_qk_norm_rope_kv8: head_dim must be 64 or 128");
    CH_REQUIRE(a->rotary_dim > 0 && a->rotary_dim % 16 == 0 && a->rotary_dim <= a->head_dim,
               "cheetah_cuda_op_qk_norm_rope_kv8: rotary_dim must be a multiple of 16 up to head_dim");
    CH_REQUIRE(a->tokens > 0 && a->tokens <= 0x7FFFFFFFu && a->max_positions > 0 && a->max_positions <= 0x7FFFFFFFu,
               "cheetah_cuda_op_qk_norm_rope_kv8: empty shape");
    CH_REQUIRE(a->q_heads > 0 && a->kv_heads > 0 && a->q_heads <= 1024 && a->kv_heads <= 1024,
               "cheetah_cuda_op_qk_norm_rope_kv8: head counts must be 1..1024");
    CH_REQUIRE(pool_in_range(a->num_pages, a->page_tokens, 1),
               "cheetah_cuda_op_qk_norm_rope_kv8: a pool holds 1 .. 2^31-1 tokens, in pages of a multiple of 16");
    const bool bf16 = a->dtype == CHEETAH_CUDA_KV_BF16;
    const size_t heads = (size_t)a->q_heads + 2 * (size_t)a->kv_heads;
    CH_REQUIRE(a->qkv_stride >= heads * a->head_dim && a->qkv_stride % (bf16 ? 8 : 4) == 0 &&
                   a->qkv_stride < ((size_t)1 << 40),
               "cheetah_cuda_op_qk_norm_rope_kv8: qkv rows must not overlap and must be 16-byte aligned");
    CH_REQUIRE(aligned(a->qkv, 16) && aligned(a->q_out, 16) && aligned(a->k_codes, 16) && aligned(a->v_codes, 16) &&
                   aligned(a->rope_cos, 16) && aligned(a->rope_sin, 16) && aligned(a->q_norm, 16) && aligned(a->k_norm, 16) &&
                   aligned(a->k_scales, 4) && aligned(a->v_scales, 4),
               "cheetah_cuda_op_qk_norm_rope_kv8: buffers must be 16-byte aligned, the scales 4-byte");
    cheetah::Kv8AppendParams p = {};
    p.q.qkv = a->qkv;
    p.q.qkv_stride = (long long)a->qkv_stride;
    p.q.q_norm = a->q_norm;
    p.q.k_norm = a->k_norm;
    p.q.eps = a->eps;
    p.q.rope_cos = a->rope_cos;
    p.q.rope_sin = a->rope_sin;
    p.q.max_positions = (int)a->max_positions;
    p.q.rotary_dim = (int)a->rotary_dim;
    p.q.positions = a->positions;
    p.q.slots = a->slots;
    p.q.tokens = (int)a->tokens;
    p.q.q_heads = (int)a->q_heads;
    p.q.kv_heads = 0;
    p.q.q_out = a->q_out;
    p.q.num_pages = (int)a->num_pages;
    p.q.page_tokens = (int)a->page_tokens;
    p.kv_heads = (int)a->kv_heads;
    p.k_codes = static_cast<uint8_t *>(a->k_codes);
    p.v_codes = static_cast<uint8_t *>(a->v_codes);
    p.k_scales = a->k_scales;
    p.v_scales = a->v_scales;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->head_dim == 64) return bf16 ? launch_append<uint16_t, 64>(p, st) : launch_append<float, 64>(p, st);
    return bf16 ? launch_append<uint16_t, 128>(p, st) : launch_append<float, 128>(p, st);
}

int cheetah_cuda_op_kv8_read(const CheetahCudaKv8Read *a, void *stream) {
    CH_REQUIRE(a != nullptr && a->k_codes && a->v_codes && a->k_scales && a->v_scales && a->slots && a->k_out && a->v_out,
               "cheetah_cuda_op_kv8_read: null argument");
    CH_REQUIRE(a->dtype == CHEETAH_CUDA_KV_BF16 || a->dtype == CHEETAH_CUDA_KV_F32, "cheetah_cuda_op_kv8_read: unknown dtype");
    CH_REQUIRE(a->head_dim == 64 || a->head_dim == 128, "cheetah_cuda_op_kv8_read: head_dim must be 64 or 128");
    CH_REQUIRE(a->tokens > 0 && a->tokens <= 0x7FFFFFFFu, "cheetah_cuda_op_kv8_read: empty shape");
    CH_REQUIRE(a->kv_heads > 0 && a->kv_heads <= 1024, "cheetah_cuda_op_kv8_read: kv_heads must be 1..1024");
    CH_REQUIRE(pool_in_range(a->num_pages, a->page_tokens, 1),
               "cheetah_cuda_op_kv8_read: a pool holds 1 .. 2^31-1 tokens, in pages of a multiple of 16");
    CH_REQUIRE(aligned(a->k_codes, 16) && aligned(a->v_codes, 16) && aligned(a->k_out, 16) && aligned(a->v_out, 16) &&
                   aligned(a->k_scales, 4) && aligned(a->v_scales, 4),
               "cheetah_cuda_op_kv8_read: buffers must be 16-byte aligned, the scales 4-byte");
    cheetah::Kv8ReadParams p = {};
    p.k_codes = static_cast<const uint8_t *>(a->k_codes);
    p.v_codes = static_cast<const uint8_t *>(a->v_codes);
    p.k_scales = a->k_scales;
    p.v_scales = a->v_scales;
    p.num_pages = (int)a->num_pages;
    p.page_tokens = (int)a->page_tokens;
    p.slots = a->slots;
    p.chunks = (long long)a->tokens * a->kv_heads * (a->head_dim / 8);
    p.kv_heads = (int)a->kv_heads;
    p.k_out = a->k_out;
    p.v_out = a->v_out;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool bf16 = a->dtype == CHEETAH_CUDA_KV_BF16;
    if (a->head_dim == 64) return bf16 ? launch_read<uint16_t, 64>(p, st) : launch_read<float, 64>(p, st);
    return bf16 ? launch_read<uint16_t, 128>(p, st) : launch_read<float, 128>(p, st);
}

// Rows of an item at most, of the kernel that takes the call. Up to 16 rows by the
// sequences' mean the keys are the products' tall side, else the rows. 32 sequences
// over 2000 to 16000 keys, heads of 128, few | many: 7 rows 58 | 75 us, 14 rows 66 |
// 75; with 32 rows to an item of the few, 28 rows took 167 | 73. The host knows `rows`
// and the batch, not how many rows each sequence has: rows behind the last sequence
// count, and a mixed batch goes by its mean. Heads as above, 4000 keys a sequence: 64
// rows of one token 62 us, with room for 64 more 73, for 128 or more 86; 256 such rows and
// a chunk of 256 403 us, in two calls 268; 64 rows and a chunk of 512 178, in two 151.
static int attention_item_rows(const CheetahCudaAttentionKv8 *a) {
    const uint64_t rows = (uint64_t)((a->rows + a->batch - 1) / a->batch) * (a->q_heads / a->kv_heads);
    return rows <= 8 ? 8 : (rows <= 16 ? 16 : 2 * cheetah::kManyRows);
}

static int check_attention_kv8(const CheetahCudaAttentionKv8 *a) {
    CH_REQUIRE(a != nullptr, "cheetah_cuda_op_attention_kv8: null argument");
    CH_REQUIRE(a->head_dim == 64 || a->head_dim == 128, "cheetah_cuda_op_attention_kv8: head_dim must be 64 or 128");
    CH_REQUIRE(a->kv_heads > 0 && a->q_heads > 0 && a->q_heads % a->kv_heads == 0 && a->q_heads / a->kv_heads <= 32 &&
                   a->q_heads <= 1024,
               "cheetah_cuda_op_attention_kv8: q_heads must be a multiple of kv_heads (group <= 32)");
    CH_REQUIRE(a->batch > 0 && a->batch <= 4096, "cheetah_cuda_op_attention_kv8: batch must be 1..4096");
    CH_REQUIRE(a->rows > 0 && a->rows <= (1u << 24), "cheetah_cuda_op_attention_kv8: rows must be 1..2^24");
    CH_REQUIRE(pool_in_range(a->num_pages, a->page_tokens, a->kv_heads) && pool_in_range(a->max_pages_per_seq, a->page_tokens, 1),
               "cheetah_cuda_op_attention_kv8: a pool holds 1 .. 2^31-1 rows of one head, a table row as many tokens, in "
               "pages of a multiple of 16");
    // The end of a key tile is counted in 31 bits too.
    CH_REQUIRE((uint64_t)a->max_pages_per_seq * a->page_tokens <= 0x7FFFFFFFull - 128,
               "cheetah_cuda_op_attention_kv8: a table row holds at most 2^31 - 129 tokens");
    CH_REQUIRE(a->sliding_window <= 0x7FFFFFFFu && a->sinks <= 0x7FFFFFFFu,
               "cheetah_cuda_op_attention_kv8: sliding_window or sinks is too large");
    // The kernel counts its cost units in 31 bits.
    const uint32_t group = a->q_heads / a->kv_heads;
    const uint64_t tiles = (uint64_t)a->max_pages_per_seq * a->page_tokens / cheetah::kKv8Keys + 1;
    const int rows = attention_item_rows(a);
    using Many = cheetah::Kv8Many<128>::Cost;
    using Few = cheetah::Kv8Few<128, 8>::Cost;
    const uint64_t nodes = rows == 2 * cheetah::kManyRows ? 2 * (cheetah::kManyRows / group) : rows / group;
    const uint64_t items = ((uint64_t)a->rows / nodes + a->batch) * a->kv_heads;
    const uint64_t units = rows == 2 * cheetah::kManyRows ? Many::TWO_TILES * tiles + Many::ITEM : Few::TWO_TILES * tiles + Few::ITEM;
    CH_REQUIRE(items * units <= 0x7FFFFFFFull, "cheetah_cuda_op_attention_kv8: too many rows and cached positions");
    return 0;
}

int cheetah_cuda_op_attention_kv8_workspace(const CheetahCudaAttentionKv8 *a, size_t *bytes) {
    CH_REQUIRE(bytes != nullptr, "cheetah_cuda_op_attention_kv8_workspace: null argument");
    if (check_attention_kv8(a) != 0) return -1;
    int device = 0;
    CH_CUDA_TRY(cudaGetDevice(&device));
    *bytes = attention_workspace(attention_ctas(device), a->head_dim).bytes;
    return 0;
}

int cheetah_cuda_op_attention_kv8(const CheetahCudaAttentionKv8 *a, void *stream) {
    if (check_attention_kv8(a) != 0) return -1;
    CH_REQUIRE(a->q && a->k_codes && a->v_codes && a->k_scales && a->v_scales && a->page_table && a->seq_lens &&
                   a->row_starts && a->out && a->workspace,
               "cheetah_cuda_op_attention_kv8: null argument");
    CH_REQUIRE(a->q_stride >= (size_t)a->q_heads * a->head_dim && a->q_stride % 8 == 0 && a->q_stride < ((size_t)1 << 32),
               "cheetah_cuda_op_attention_kv8: q rows must not overlap and must be 16-byte aligned");
    CH_REQUIRE(aligned(a->q, 16) && aligned(a->k_codes, 16) && aligned(a->v_codes, 16) && aligned(a->out, 16) &&
                   aligned(a->k_scales, 4) && aligned(a->v_scales, 4) && aligned(a->workspace, 256),
               "cheetah_cuda_op_attention_kv8: q, out and the codes must be 16-byte aligned, the scales 4-byte, the workspace "
               "256-byte");
    int device = 0;
    CH_CUDA_TRY(cudaGetDevice(&device));
    const int ctas = attention_ctas(device);
    const AttentionWorkspace w = attention_workspace(ctas, a->head_dim);
    CH_REQUIRE(a->workspace_bytes >= w.bytes,
               "cheetah_cuda_op_attention_kv8: the workspace holds " + std::to_string(a->workspace_bytes) + " of " +
                   std::to_string(w.bytes) + " bytes");
    cheetah::Kv8AttnParams p = {};
    p.q = static_cast<const uint16_t *>(a->q);
    p.q_stride = (long long)a->q_stride;
    p.k_codes = static_cast<const uint8_t *>(a->k_codes);
    p.v_codes = static_cast<const uint8_t *>(a->v_codes);
    p.k_scales = a->k_scales;
    p.v_scales = a->v_scales;
    p.page_table = a->page_table;
    p.max_pages = (int)a->max_pages_per_seq;
    p.num_pages = (int)a->num_pages;
    p.page_tokens = (int)a->page_tokens;
    p.seq_lens = a->seq_lens;
    p.row_starts = a->row_starts;
    p.batch = (int)a->batch;
    p.rows = (int)a->rows;
    p.window = (int)a->sliding_window;
    p.sinks = (int)a->sinks;
    p.q_heads = (int)a->q_heads;
    p.kv_heads = (int)a->kv_heads;
    p.scale_log2 = 1.4426950408889634f / sqrtf((float)a->head_dim);
    p.out = static_cast<uint16_t *>(a->out);
    p.group = (int)(a->q_heads / a->kv_heads);
    p.box_shift = a->page_tokens % 128 == 0 ? 7 : (a->page_tokens % 64 == 0 ? 6 : (a->page_tokens % 32 == 0 ? 5 : 4));
    uint8_t *ws = static_cast<uint8_t *>(a->workspace);
    p.splits = reinterpret_cast<cheetah::TreeSplit *>(ws + w.splits);
    p.part_ml = reinterpret_cast<float2 *>(ws + w.ml);
    p.part_o = reinterpret_cast<float *>(ws + w.o);
    CUtensorMap k_map, v_map;
    const uint64_t pool_rows = (uint64_t)a->num_pages * a->kv_heads * a->page_tokens;
    if (make_codes_map(&k_map, a->k_codes, pool_rows, a->head_dim, 1u << p.box_shift) != 0 ||
        make_codes_map(&v_map, a->v_codes, pool_rows, a->head_dim, 1u << p.box_shift) != 0) {
        return -1;
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int rows = attention_item_rows(a);
    if (a->head_dim == 64) {
        return rows == 8    ? launch_attention_few<64, 8>(k_map, v_map, p, device, ctas, st)
               : rows == 16 ? launch_attention_few<64, 16>(k_map, v_map, p, device, ctas, st)
                            : launch_attention_many<64>(k_map, v_map, p, device, ctas, st);
    }
    return rows == 8    ? launch_attention_few<128, 8>(k_map, v_map, p, device, ctas, st)
           : rows == 16 ? launch_attention_few<128, 16>(k_map, v_map, p, device, ctas, st)
                        : launch_attention_many<128>(k_map, v_map, p, device, ctas, st);
}

int cheetah_cuda_op_verify_drafts(const CheetahCudaVerifyDrafts *a, void *stream) {
    CH_REQUIRE(a != nullptr && a->target_probs && a->tokens && a->row_starts && a->accept_u && a->sample_u && a->accepted &&
                   a->out_tokens,
               "cheetah_cuda_op_verify_drafts: null argument");
    // (Rows are walked in steps of up to a block, in 31 bits.)
    CH_REQUIRE(a->rows > 0 && a->rows <= (1u << 30) && a->vocab > 0 && a->vocab <= (1u << 30),
               "cheetah_cuda_op_verify_drafts: rows and vocab must be 1..2^30");
    CH_REQUIRE(a->batch > 0 && a->batch <= 65535, "cheetah_cuda_op_verify_drafts: batch must be 1..65535");
    CH_REQUIRE((a->target_stride >= a->vocab || a->rows == 1) && a->target_stride < ((size_t)1 << 40) &&
                   (a->draft_probs == nullptr ||
                    ((a->draft_stride >= a->vocab || a->rows == 1) && a->draft_stride < ((size_t)1 << 40))),
               "cheetah_cuda_op_verify_drafts: rows must not overlap");
    CH_REQUIRE(aligned(a->target_probs, 4) && aligned(a->draft_probs, 4),
               "cheetah_cuda_op_verify_drafts: probabilities must be aligned to their type");
    // CTAs of a sequence read its tokens while one writes what it kept.
    CH_REQUIRE(a->out_tokens + a->rows <= a->tokens || a->tokens + a->rows <= a->out_tokens,
               "cheetah_cuda_op_verify_drafts: out_tokens must not overlap tokens");
    cheetah::VerifyDraftsParams p = {};
    p.target = a->target_probs;
    p.draft = a->draft_probs;
    p.target_stride = (long long)a->target_stride;
    p.draft_stride = (long long)a->draft_stride;
    p.rows = (int)a->rows;
    p.vocab = (int)a->vocab;
    p.tokens = a->tokens;
    p.row_starts = a->row_starts;
    p.batch = (int)a->batch;
    p.accept_u = a->accept_u;
    p.sample_u = a->sample_u;
    p.accepted = a->accepted;
    p.out_tokens = a->out_tokens;
    int device = 0;
    CH_CUDA_TRY(cudaGetDevice(&device));
    // Parts of a row: as many as run at once, each with two chunks at least. CTAs
    // that wait for others to end cost more than thinner ones gain: 96 sequences over
    // 152064 tokens take 23.3 us in 384 CTAs and 29.4 us in 768 (444 run at once), 300
    // over 32000 take 20.0 us in 300 and 21.7 us in 600.
    const long long vecs = ((long long)a->vocab + 6) / 4;
    p.parts = 1;
    while (p.parts < cheetah::kVdMaxCluster && 2ll * a->batch * p.parts <= (long long)cheetah::kVdResident * cheetah::sm_count(device) &&
           vecs >= 4ll * p.parts * cheetah::kVdThreads) {
        p.parts *= 2;
    }
    p.chunk_vecs = cheetah::kVdThreads;
    while ((vecs + p.chunk_vecs - 1) / p.chunk_vecs > (long long)cheetah::kVdMaxChunks * p.parts) p.chunk_vecs *= 2;
    auto kernel = cheetah::verify_drafts_kernel;
    if (p.parts > 8) CH_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(a->batch * (uint32_t)p.parts));
    config.blockDim = dim3(cheetah::kVdThreads);
    config.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)p.parts;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = 2;
    CH_CUDA_TRY(cudaLaunchKernelEx(&config, kernel, p));
    return 0;
}

}  // extern "C"
