// Host launchers of the tree-speculation kernels (raw pointers + stream).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace cb {

// Layout of one tree step on the device: request b owns node rows [cu[b], cu[b+1]); its position p is cached in slot
// table[b * P + p / page] * page + p % page; node i of it sits at position ctx[b] + i.
struct TreeLayout {
  const int* cu;           // [B + 1]
  const int* ctx;          // [B]
  const int* table;        // [B, P]
  int B, P, page;
};

// q [T, H, D] (bf16; fp16 for fp8 rows), kv rows [S, row bytes], mask [T] (bit j: the node sees node j), req [T]
// -> out [T, H, 512] bf16
cudaError_t tree_mla(const void* q, int T, int H, int D, bool f8, const void* kv, const TreeLayout& lay,
                     const int64_t* mask, const int* req, float scale, const float* sink, void* out, cudaStream_t s);

// logits [T, ld] fp32 or bf16, draft [T, V] fp32 or null -> path, tokens [B, N], n_accepted [B], logprobs [B, N]
cudaError_t tree_verify(const void* logits, bool bf16, int64_t ld, int V, const int* tokens, const int* cu,
                        const int* parent, int B, int N, const float* uniforms, const float* noise,
                        const float* temperature, const float* draft, int* path, int* n_accepted, int* out_tokens,
                        float* logprobs, cudaStream_t s);

// caches: [n, 2] int64 (address, row bytes); max_row: the largest row; wide: every address and row is a multiple of 16
// bytes (of 4 otherwise)
cudaError_t tree_commit(const int64_t* caches, int n, int max_row, bool wide, const TreeLayout& lay, int N, const int* path,
                        const int* n_accepted, cudaStream_t s);

}  // namespace cb
