// An entry for the tests to the joins of the 8-bit cache's attention alone: what
// they do after a CTA whose wait gave up cannot be reached through the library
// without making a wait run out.
#include <cuda.h>
#include <cuda_runtime.h>

#include "attention_kv8.cuh"

// splits: one per CTA of the attention launch; out: bf16 [rows][q_heads][64].
extern "C" __attribute__((visibility("default"))) int kv8_join(const int *parts, int ctas, const int32_t *row_starts, int batch,
                                                              int rows, int q_heads, void *splits, void *out, void *stream) {
    if (ctas < 1 || ctas > cheetah::kKv8MaxCtas) return -1;
    cheetah::TreeSplit host[cheetah::kKv8MaxCtas] = {};
    for (int i = 0; i < ctas; ++i) host[i].parts = parts[i];
    cheetah::Kv8AttnParams p = {};
    p.row_starts = row_starts;
    p.batch = batch;
    p.rows = rows;
    p.q_heads = q_heads;
    p.group = 1;
    p.splits = static_cast<cheetah::TreeSplit *>(splits);
    p.out = static_cast<uint16_t *>(out);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (cudaMemcpyAsync(splits, host, ctas * sizeof(host[0]), cudaMemcpyHostToDevice, st) != cudaSuccess) return -2;
    cheetah::kv8_merge_kernel<64, 16><<<dim3(ctas, 16 / cheetah::kKv8MergeRows), cheetah::kKv8MergeThreads, 0, st>>>(p, ctas);
    return cudaGetLastError() == cudaSuccess ? 0 : -3;
}
