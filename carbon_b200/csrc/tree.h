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

// Work of one attention call, made by tree_schedule: a CTA pair runs the items [first[c], first[c + 1]) one after the
// other.  An item is one 128-row tile (rows = nodes x heads of one request) over a range of 128-key tiles.
struct alignas(16) TreeItem {
  int b, row, tile, n_tiles;
  int part;                // partial-result slot, -1 = the whole row tile
  int ctx, c0, n;          // the request's cached tokens, first node row and nodes
};
// A row tile whose partial results [part, part + n) are merged; its request's first node row and nodes x heads rows.
struct alignas(8) TreeMerge { int row, part, n, c0, rows, pad; };
struct TreeWork {
  const int* first;        // [clusters + 1]
  const TreeItem* items;
  const TreeMerge* merges;
  int clusters, n_merges, most_parts;     // most_parts: of one row tile
  // 128-row blocks of the staging buffer, one per whole key tile before the tree: (request, key tile), and each
  // request's first block
  const int2* stage;
  const int* stage_at;     // [B]
  int n_stage;
};

// q [T, H, D] (bf16; fp16 for fp8 rows), kv rows [S, row bytes], mask [T] (bit j: the node sees node j)
// -> out [T, H, 512] bf16.  part_o [parts, 128, 512], part_ml [parts, 128, 2]: workspaces; staged: null, or
// [n_stage * 128, D] 16-bit, where whole key tiles are first expanded to dense rows.
cudaError_t tree_mla(const void* q, int T, int H, int D, bool f8, const void* kv, int64_t S, const TreeLayout& lay,
                     const TreeWork& work, const int64_t* mask, float scale, const float* sink, float* part_o,
                     float* part_ml, void* staged, int* status, void* out, cudaStream_t s);
// CTA pairs of the attention kernel that fit on the current device at once
int tree_mla_clusters();

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
