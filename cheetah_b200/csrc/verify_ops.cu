// The op entries of a step that verifies drafted tokens (include/cheetah_cuda.h):
// page slots, q/k norm with rotation and cache append, tree attention, token
// log probabilities. Each checks its arguments, launches on the caller's
// stream and keeps nothing.
#include <cuda.h>
#include <cuda_runtime.h>
#include <math.h>

#include <algorithm>
#include <atomic>
#include <string>
#include <type_traits>

#include "cheetah_cuda.h"
#include "common.cuh"
#include "launch.cuh"
#include "page_slots.cuh"
#include "qk_norm_rope.cuh"
#include "token_logprobs.cuh"
#include "tree_attention.cuh"

using cheetah::launch_ex;

namespace {

bool aligned(const void *p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

// A pool's slots are numbered in 32 bits.
bool pool_in_range(uint32_t num_pages, uint32_t page_tokens) {
    return num_pages > 0 && page_tokens > 0 && (uint64_t)num_pages * page_tokens <= 0x7FFFFFFFull;
}

// 2D map over a bf16 pool viewed as [rows][head_dim]: 64-column boxes of
// `box_rows` rows of one page, 128-byte swizzle.
int make_pool_map(CUtensorMap *map, const void *base, uint64_t rows, uint32_t head_dim, uint32_t box_rows) {
    auto encode = cheetah::tensor_map_encoder();
    CH_REQUIRE(encode != nullptr, "CUDA backend: cuTensorMapEncodeTiled is unavailable");
    cuuint64_t dims[2] = {head_dim, rows};
    cuuint64_t strides[1] = {(cuuint64_t)head_dim * 2};
    cuuint32_t box[2] = {64u, box_rows};
    cuuint32_t estr[2] = {1u, 1u};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void *>(base), dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    CH_REQUIRE(r == CUDA_SUCCESS, "CUDA backend: cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")");
    return 0;
}

// 3D map over q [rows][q_heads][head_dim]: boxes of 64 columns, the heads of
// one KV group and the nodes of a Q tile. Rows past the end read as zero.
int make_q_map(CUtensorMap *map, const CheetahCudaTreeAttention &a, uint32_t group, uint32_t tile_nodes) {
    auto encode = cheetah::tensor_map_encoder();
    CH_REQUIRE(encode != nullptr, "CUDA backend: cuTensorMapEncodeTiled is unavailable");
    cuuint64_t dims[3] = {a.head_dim, a.q_heads, a.rows};
    cuuint64_t strides[2] = {(cuuint64_t)a.head_dim * 2, (cuuint64_t)a.q_stride * 2};
    cuuint32_t box[3] = {64u, group, tile_nodes};
    cuuint32_t estr[3] = {1u, 1u, 1u};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(a.q), dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    CH_REQUIRE(r == CUDA_SUCCESS, "CUDA backend: cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")");
    return 0;
}

// Warps of a q/k norm call: a warp walks over a whole row where there are some
// 48 head groups per SM (its cos/sin and weights are then read once), over one
// group of heads where there are fewer and latency counts. 9 groups a row: 256
// rows take 5.3 us whole and 2.7 in groups, 1021 rows 6.2 and 7.1, 4096 rows 17
// and 30; 3 groups a row: 2048 rows 5.9 and 5.1, 4096 rows 6.2 and 9.1. Rows of
// up to 3 groups have all their loads in flight with fewer registers (16384 of
// them 23 us, with room for 5 groups 30).
template <typename TIN, int HD>
int launch_qk(cheetah::QkNormRopeParams p, bool kv_bf16, cudaStream_t stream) {
    constexpr int kHeads = cheetah::kWarp / (HD / 2 / (16 / (int)sizeof(TIN)));
    const int steps = (p.q_heads + 2 * p.kv_heads + kHeads - 1) / kHeads;
    int device = 0;
    CH_CUDA_TRY(cudaGetDevice(&device));
    p.steps = (long long)p.tokens * steps >= 48ll * cheetah::sm_count(device) ? steps : 1;
    p.row_units = (steps + p.steps - 1) / p.steps;
    const uint64_t blocks = ((uint64_t)p.tokens * p.row_units + cheetah::kQkWarps - 1) / cheetah::kQkWarps;
    CH_REQUIRE(blocks <= 0x7FFFFFFFull, "cheetah_cuda_op_qk_norm_rope: too many rows");
    auto pick = [&](auto u) {
        constexpr int U = decltype(u)::value;
        return kv_bf16 ? cheetah::qk_norm_rope_rows_kernel<TIN, uint16_t, HD, U> : cheetah::qk_norm_rope_rows_kernel<TIN, float, HD, U>;
    };
    auto kernel = p.steps == 1  ? pick(std::integral_constant<int, 1>())
                  : p.steps <= 3 ? pick(std::integral_constant<int, 3>())
                                 : pick(std::integral_constant<int, cheetah::kQkUnroll>());
    CH_CUDA_TRY(launch_ex(kernel, dim3((unsigned)blocks), dim3(cheetah::kQkWarps * cheetah::kWarp), 0, stream, true, p));
    return 0;
}

// A cluster of CTAs per row: the number that leaves the busiest SM the least
// (rows divide badly among 148 SMs, and one row fills 16). A part is charged 3%
// for its join, 20% where it sorts too, and holds at least half a sample: 500
// bf16 rows of 152064 take 37.5 us in two parts and 39.6 in one without
// alternatives, 59.2 and 55.4 with twenty.
int launch_logprobs(const cheetah::LogprobParams &p, bool bf16, cudaStream_t stream) {
    auto kernel = bf16 ? cheetah::token_logprobs_kernel<uint16_t> : cheetah::token_logprobs_kernel<float>;
    int device = 0;
    CH_CUDA_TRY(cudaGetDevice(&device));
    const long long sms = cheetah::sm_count(device);
    const int sample = cheetah::kLpThreads * cheetah::kLpLoads * (bf16 ? 8 : 4);
    int parts = 1;
    double least = 0.0;
    for (int n = 1; n <= cheetah::kLpMaxCluster && (n == 1 || p.vocab / n >= sample / 2); n *= 2) {
        const long long busiest = ((long long)p.rows * n + sms - 1) / sms;
        const double cost = (double)busiest / n * (1.0 + (p.top > 0 ? 0.2 : 0.03) * n);
        if (n == 1 || cost < least) {
            least = cost;
            parts = n;
        }
    }
    CH_REQUIRE((uint64_t)p.rows * parts <= 0x7FFFFFFFull, "cheetah_cuda_op_token_logprobs: too many rows");
    if (parts > 8) CH_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(p.rows * parts));
    config.blockDim = dim3(cheetah::kLpThreads);
    config.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)parts;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = 2;
    CH_CUDA_TRY(cudaLaunchKernelEx(&config, kernel, p));
    return 0;
}

int tree_ctas(int device) { return std::min(cheetah::sm_count(device), cheetah::kTreeMaxCtas); }

// Workspace of a tree attention call of `ctas` CTAs.
struct TreeWorkspace {
    size_t splits, ml, o, bytes;
};
TreeWorkspace tree_workspace(int ctas, uint32_t head_dim) {
    auto up = [](size_t x) { return (x + 255) & ~size_t(255); };
    TreeWorkspace w;
    w.splits = 0;
    w.ml = up(ctas * sizeof(cheetah::TreeSplit));
    w.o = w.ml + up((size_t)ctas * 512 * sizeof(float2));
    w.bytes = w.o + (size_t)ctas * 512 * head_dim * sizeof(float);
    return w;
}

// Up to this many rows of all heads (four Q tiles) the exact products are used:
// 8 nodes of 14 heads at 708 keys take 12.9 us with them and 12.1 without; 32
// sequences of up to 16 nodes of 28 heads would take 75 us instead of 65.
constexpr uint64_t kTreeExactRows = 512;

template <int HD, bool REST>
int launch_tree_attention(const CUtensorMap &q_map, const CUtensorMap &k_map, const CUtensorMap &v_map,
                          const cheetah::TreeAttnParams &p, int device, int ctas, cudaStream_t stream) {
    static std::atomic<uint64_t> done{0};
    constexpr size_t smem = cheetah::tree_attention_smem<HD>();
    CH_CUDA_TRY(cheetah::allow_smem(cheetah::tree_attention_kernel<HD, REST>, smem, device, done));
    CH_CUDA_TRY(launch_ex(cheetah::tree_attention_kernel<HD, REST>, dim3(ctas), dim3(cheetah::kTreeThreads), smem, stream, true,
                          q_map, k_map, v_map, p));
    CH_CUDA_TRY(launch_ex(cheetah::tree_merge_kernel<HD>, dim3(ctas * cheetah::kTreeMergeCtas), dim3(cheetah::kTreeMergeThreads),
                          0, stream, true, p, ctas));
    return 0;
}

}  // namespace

extern "C" {

int cheetah_cuda_op_page_slots(const CheetahCudaPageSlots *a, void *stream) {
    CH_REQUIRE(a != nullptr && a->cached && a->new_tokens && a->free_count && a->page_table && a->row_starts &&
                   a->seq_lens && a->positions && a->seq_ids && a->slots && a->counts,
               "cheetah_cuda_op_page_slots: null argument");
    CH_REQUIRE(a->free_pages != nullptr || a->free_capacity == 0, "cheetah_cuda_op_page_slots: null free list");
    CH_REQUIRE(a->batch > 0 && a->batch <= (uint32_t)cheetah::kSlotMaxBatch,
               "cheetah_cuda_op_page_slots: batch must be 1.." + std::to_string(cheetah::kSlotMaxBatch));
    CH_REQUIRE(a->max_tokens > 0 && a->max_tokens <= 0x7FFFFFFFu && a->free_capacity <= 0x7FFFFFFFu,
               "cheetah_cuda_op_page_slots: max_tokens must be positive, and lengths below 2^31");
    CH_REQUIRE(pool_in_range(a->num_pages, a->page_tokens) && pool_in_range(a->max_pages_per_seq, a->page_tokens),
               "cheetah_cuda_op_page_slots: a pool and a table row hold 1 .. 2^31-1 tokens");
    int device = 0;
    CH_CUDA_TRY(cudaGetDevice(&device));
    cheetah::PageSlotParams p = {};
    p.cached = a->cached;
    p.new_tokens = a->new_tokens;
    p.free_pages = a->free_pages;
    p.free_count = a->free_count;
    p.free_capacity = (int)a->free_capacity;
    p.batch = (int)a->batch;
    p.page_table = a->page_table;
    p.max_pages = (int)a->max_pages_per_seq;
    p.num_pages = (int)a->num_pages;
    p.page_tokens = (int)a->page_tokens;
    p.max_tokens = (int)a->max_tokens;
    p.row_starts = a->row_starts;
    p.seq_lens = a->seq_lens;
    p.positions = a->positions;
    p.seq_ids = a->seq_ids;
    p.slots = a->slots;
    p.counts = a->counts;
    const size_t smem = (size_t)a->batch * 3 * sizeof(int32_t);
    // Four rows per thread once one per thread would take several CTAs of
    // every SM (4.1 us against 5.9 for 541 rows, 19 against 12.8 for 10^6).
    const bool wide = (long long)p.max_tokens > 2ll * cheetah::sm_count(device) * cheetah::kSlotThreads;
    const int vec = wide && aligned(a->positions, 16) && aligned(a->seq_ids, 16) && aligned(a->slots, 16) ? 4 : 1;
    auto kernel = vec == 4 ? cheetah::page_slots_kernel<4> : cheetah::page_slots_kernel<1>;
    if (smem > 48 * 1024) {
        // What the largest batch needs, whatever this one does: the limit
        // belongs to the kernel, and another thread may be about to launch it.
        static std::atomic<uint64_t> done[2];
        CH_CUDA_TRY(cheetah::allow_smem(kernel, (size_t)cheetah::kSlotMaxBatch * 3 * sizeof(int32_t), device, done[vec == 4]));
    }
    const int per_block = cheetah::kSlotThreads * vec;
    const int blocks = (int)std::min<long long>(2 * cheetah::sm_count(device), ((long long)p.max_tokens + per_block - 1) / per_block);
    CH_CUDA_TRY(launch_ex(kernel, dim3(blocks), dim3(cheetah::kSlotThreads), smem, static_cast<cudaStream_t>(stream), true, p));
    return 0;
}

int cheetah_cuda_op_qk_norm_rope(const CheetahCudaQkNormRope *a, void *stream) {
    CH_REQUIRE(a != nullptr && a->qkv && a->rope_cos && a->rope_sin && a->positions && a->slots && a->q_out &&
                   a->k_pool && a->v_pool,
               "cheetah_cuda_op_qk_norm_rope: null argument");
    CH_REQUIRE((a->dtype == CHEETAH_CUDA_KV_BF16 || a->dtype == CHEETAH_CUDA_KV_F32) &&
                   (a->kv_dtype == CHEETAH_CUDA_KV_BF16 || a->kv_dtype == CHEETAH_CUDA_KV_F32),
               "cheetah_cuda_op_qk_norm_rope: unknown dtype");
    CH_REQUIRE(a->head_dim == 64 || a->head_dim == 128, "cheetah_cuda_op_qk_norm_rope: head_dim must be 64 or 128");
    CH_REQUIRE(a->rotary_dim > 0 && a->rotary_dim % 16 == 0 && a->rotary_dim <= a->head_dim,
               "cheetah_cuda_op_qk_norm_rope: rotary_dim must be a multiple of 16 up to head_dim");
    CH_REQUIRE(a->tokens > 0 && a->tokens <= 0x7FFFFFFFu && a->max_positions > 0 && a->max_positions <= 0x7FFFFFFFu,
               "cheetah_cuda_op_qk_norm_rope: empty shape");
    CH_REQUIRE(a->q_heads > 0 && a->kv_heads > 0 && a->q_heads <= 1024 && a->kv_heads <= 1024,
               "cheetah_cuda_op_qk_norm_rope: head counts must be 1..1024");
    CH_REQUIRE(pool_in_range(a->num_pages, a->page_tokens),
               "cheetah_cuda_op_qk_norm_rope: a pool holds 1 .. 2^31-1 tokens");
    const bool bf16 = a->dtype == CHEETAH_CUDA_KV_BF16;
    const size_t heads = (size_t)a->q_heads + 2 * (size_t)a->kv_heads;
    CH_REQUIRE(a->qkv_stride >= heads * a->head_dim && a->qkv_stride % (bf16 ? 8 : 4) == 0 &&
                   a->qkv_stride < ((size_t)1 << 40),
               "cheetah_cuda_op_qk_norm_rope: qkv rows must not overlap and must be 16-byte aligned");
    CH_REQUIRE(aligned(a->qkv, 16) && aligned(a->q_out, 16) && aligned(a->k_pool, 16) && aligned(a->v_pool, 16) &&
                   aligned(a->rope_cos, 16) && aligned(a->rope_sin, 16) && aligned(a->q_norm, 16) && aligned(a->k_norm, 16),
               "cheetah_cuda_op_qk_norm_rope: buffers must be 16-byte aligned");
    cheetah::QkNormRopeParams p = {};
    p.qkv = a->qkv;
    p.qkv_stride = (long long)a->qkv_stride;
    p.q_norm = a->q_norm;
    p.k_norm = a->k_norm;
    p.eps = a->eps;
    p.rope_cos = a->rope_cos;
    p.rope_sin = a->rope_sin;
    p.max_positions = (int)a->max_positions;
    p.rotary_dim = (int)a->rotary_dim;
    p.positions = a->positions;
    p.slots = a->slots;
    p.tokens = (int)a->tokens;
    p.q_heads = (int)a->q_heads;
    p.kv_heads = (int)a->kv_heads;
    p.q_out = a->q_out;
    p.k_pool = a->k_pool;
    p.v_pool = a->v_pool;
    p.num_pages = (int)a->num_pages;
    p.page_tokens = (int)a->page_tokens;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool kv_bf16 = a->kv_dtype == CHEETAH_CUDA_KV_BF16;
    if (a->head_dim == 64) return bf16 ? launch_qk<uint16_t, 64>(p, kv_bf16, st) : launch_qk<float, 64>(p, kv_bf16, st);
    return bf16 ? launch_qk<uint16_t, 128>(p, kv_bf16, st) : launch_qk<float, 128>(p, kv_bf16, st);
}

static int check_tree_attention(const CheetahCudaTreeAttention *a) {
    CH_REQUIRE(a != nullptr, "cheetah_cuda_op_tree_attention: null argument");
    CH_REQUIRE(a->head_dim == 64 || a->head_dim == 128, "cheetah_cuda_op_tree_attention: head_dim must be 64 or 128");
    CH_REQUIRE(a->kv_heads > 0 && a->q_heads > 0 && a->q_heads % a->kv_heads == 0 && a->q_heads / a->kv_heads <= 32 &&
                   a->q_heads <= 1024,
               "cheetah_cuda_op_tree_attention: q_heads must be a multiple of kv_heads (group <= 32)");
    CH_REQUIRE(a->batch > 0 && a->batch <= 4096, "cheetah_cuda_op_tree_attention: batch must be 1..4096");
    CH_REQUIRE(a->rows > 0 && a->rows <= (1u << 24), "cheetah_cuda_op_tree_attention: rows must be 1..2^24");
    CH_REQUIRE(a->page_tokens > 0 && a->page_tokens % 16 == 0,
               "cheetah_cuda_op_tree_attention: page_tokens must be a multiple of 16");
    CH_REQUIRE(pool_in_range(a->num_pages, a->page_tokens) && pool_in_range(a->max_pages_per_seq, a->page_tokens) &&
                   (uint64_t)a->num_pages * a->kv_heads * a->page_tokens <= 0x7FFFFFFFull,
               "cheetah_cuda_op_tree_attention: a pool holds 1 .. 2^31-1 rows of one head, a table row as many tokens");
    // The end of a key tile is counted in 31 bits too.
    CH_REQUIRE((uint64_t)a->max_pages_per_seq * a->page_tokens <= 0x7FFFFFFFull - cheetah::kTreeKeys,
               "cheetah_cuda_op_tree_attention: a table row holds at most 2^31 - 129 tokens");
    CH_REQUIRE(a->mask_words > 0 && a->mask_words <= 16, "cheetah_cuda_op_tree_attention: mask_words must be 1..16");
    CH_REQUIRE(a->sliding_window <= 0x7FFFFFFFu, "cheetah_cuda_op_tree_attention: sliding_window is too large");
    // The kernel counts its cost units (at most 4 per key tile of an item, and
    // 8 per item) in 31 bits.
    const uint64_t tile_rows = 2 * (cheetah::kTreeRows / (a->q_heads / a->kv_heads));
    const uint64_t items = ((uint64_t)a->rows / tile_rows + a->batch + 1) * a->kv_heads;
    const uint64_t tiles = (uint64_t)a->max_pages_per_seq * a->page_tokens / cheetah::kTreeKeys + 1;
    CH_REQUIRE(items * (4 * tiles + 8) <= 0x7FFFFFFFull, "cheetah_cuda_op_tree_attention: too many rows and cached positions");
    return 0;
}

int cheetah_cuda_op_tree_attention_workspace(const CheetahCudaTreeAttention *a, size_t *bytes) {
    CH_REQUIRE(bytes != nullptr, "cheetah_cuda_op_tree_attention_workspace: null argument");
    if (check_tree_attention(a) != 0) return -1;
    int device = 0;
    CH_CUDA_TRY(cudaGetDevice(&device));
    *bytes = tree_workspace(tree_ctas(device), a->head_dim).bytes;
    return 0;
}

int cheetah_cuda_op_tree_attention(const CheetahCudaTreeAttention *a, void *stream) {
    if (check_tree_attention(a) != 0) return -1;
    CH_REQUIRE(a->q && a->k_pool && a->v_pool && a->page_table && a->seq_lens && a->row_starts && a->tree_mask && a->out &&
                   a->workspace,
               "cheetah_cuda_op_tree_attention: null argument");
    CH_REQUIRE(a->sliding_window == 0 || a->positions != nullptr,
               "cheetah_cuda_op_tree_attention: a sliding window needs the rows' positions");
    CH_REQUIRE(a->q_stride >= (size_t)a->q_heads * a->head_dim && a->q_stride % 8 == 0 && a->q_stride < ((size_t)1 << 32),
               "cheetah_cuda_op_tree_attention: q rows must not overlap and must be 16-byte aligned");
    CH_REQUIRE(aligned(a->q, 16) && aligned(a->k_pool, 16) && aligned(a->v_pool, 16) && aligned(a->out, 16) &&
                   aligned(a->tree_mask, 8) && aligned(a->workspace, 256),
               "cheetah_cuda_op_tree_attention: q, out and the pools must be 16-byte aligned, the mask 8-byte, the "
               "workspace 256-byte");
    int device = 0;
    CH_CUDA_TRY(cudaGetDevice(&device));
    const int ctas = tree_ctas(device);
    const TreeWorkspace w = tree_workspace(ctas, a->head_dim);
    CH_REQUIRE(a->workspace_bytes >= w.bytes,
               "cheetah_cuda_op_tree_attention: the workspace holds " + std::to_string(a->workspace_bytes) + " of " +
                   std::to_string(w.bytes) + " bytes");
    const uint32_t group = a->q_heads / a->kv_heads;
    cheetah::TreeAttnParams p = {};
    p.page_table = a->page_table;
    p.max_pages = (int)a->max_pages_per_seq;
    p.num_pages = (int)a->num_pages;
    p.page_tokens = (int)a->page_tokens;
    p.box_keys = a->page_tokens % 64 == 0 ? 64 : (a->page_tokens % 32 == 0 ? 32 : 16);
    p.seq_lens = a->seq_lens;
    p.row_starts = a->row_starts;
    p.batch = (int)a->batch;
    p.rows = (int)a->rows;
    p.tree_mask = reinterpret_cast<const uint32_t *>(a->tree_mask);
    p.mask_words32 = 2 * (int)a->mask_words;
    p.positions = a->positions;
    p.window = (int)a->sliding_window;
    p.q_heads = (int)a->q_heads;
    p.kv_heads = (int)a->kv_heads;
    p.group = (int)group;
    p.tile_nodes = cheetah::kTreeRows / (int)group;
    p.scale_log2 = 1.4426950408889634f / sqrtf((float)a->head_dim);
    p.v_pool = static_cast<const uint16_t *>(a->v_pool);
    p.out = static_cast<uint16_t *>(a->out);
    uint8_t *ws = static_cast<uint8_t *>(a->workspace);
    p.splits = reinterpret_cast<cheetah::TreeSplit *>(ws + w.splits);
    p.part_ml = reinterpret_cast<float2 *>(ws + w.ml);
    p.part_o = reinterpret_cast<float4 *>(ws + w.o);
    CUtensorMap q_map, k_map, v_map;
    const uint64_t rows = (uint64_t)a->num_pages * a->kv_heads * a->page_tokens;
    if (make_q_map(&q_map, *a, group, (uint32_t)p.tile_nodes) != 0 ||
        make_pool_map(&k_map, a->k_pool, rows, a->head_dim, (uint32_t)p.box_keys) != 0 ||
        make_pool_map(&v_map, a->v_pool, rows, a->head_dim, (uint32_t)p.box_keys) != 0) {
        return -1;
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool exact = (uint64_t)a->rows * a->q_heads <= kTreeExactRows;
    auto launch = a->head_dim == 64 ? (exact ? launch_tree_attention<64, true> : launch_tree_attention<64, false>)
                                    : (exact ? launch_tree_attention<128, true> : launch_tree_attention<128, false>);
    return launch(q_map, k_map, v_map, p, device, ctas, st);
}

int cheetah_cuda_op_token_logprobs(const CheetahCudaTokenLogprobs *a, void *stream) {
    CH_REQUIRE(a != nullptr && a->logits && a->tokens && a->logprob, "cheetah_cuda_op_token_logprobs: null argument");
    CH_REQUIRE(a->dtype == CHEETAH_CUDA_KV_BF16 || a->dtype == CHEETAH_CUDA_KV_F32,
               "cheetah_cuda_op_token_logprobs: unknown dtype");
    CH_REQUIRE(a->rows > 0 && a->rows <= 0x7FFFFFFFu && a->vocab > 0, "cheetah_cuda_op_token_logprobs: empty shape");
    // Ids and vector numbers are stepped through in 32 bits.
    CH_REQUIRE(a->vocab <= (1u << 30), "cheetah_cuda_op_token_logprobs: vocab must be at most 2^30");
    CH_REQUIRE(a->top <= (uint32_t)cheetah::kLpMaxTop && a->top <= a->vocab,
               "cheetah_cuda_op_token_logprobs: top must be at most 32 and at most vocab");
    CH_REQUIRE(a->top == 0 || (a->top_ids && a->top_logprobs),
               "cheetah_cuda_op_token_logprobs: top needs top_ids and top_logprobs");
    CH_REQUIRE((a->row_stride >= a->vocab || a->rows == 1) && a->row_stride < ((size_t)1 << 40),
               "cheetah_cuda_op_token_logprobs: rows must not overlap");
    const bool bf16 = a->dtype == CHEETAH_CUDA_KV_BF16;
    CH_REQUIRE(aligned(a->logits, bf16 ? 2 : 4), "cheetah_cuda_op_token_logprobs: logits must be aligned to their type");
    cheetah::LogprobParams p = {};
    p.logits = a->logits;
    p.row_stride = (long long)a->row_stride;
    p.rows = (int)a->rows;
    p.vocab = (int)a->vocab;
    p.tokens = a->tokens;
    p.top = (int)a->top;
    p.logprob = a->logprob;
    p.rank = a->rank;
    p.entropy = a->entropy;
    p.top_ids = a->top_ids;
    p.top_logprobs = a->top_logprobs;
    return launch_logprobs(p, bf16, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
