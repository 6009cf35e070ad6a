// Verification of drafted token trees against the target's probabilities, and the commit of the accepted branch.
//
// Verification walks each request's tree from the root.  At node v with target probabilities p = softmax(l_v / T) the
// remainder r starts as p; child c (index order) is accepted when u_c q(x_c) < r(x_c), q the distribution its token was
// drawn from; a rejection leaves r <- max(r - q, 0) / (its sum).  Where no child is accepted the next token is
// argmax_i r_i / e_i with e ~ Exp(1) given, which is a draw from r.  Sums, maxima and probabilities are fp32.
#include "common.cuh"
#include "tree.h"

namespace cb {
namespace tree {

constexpr int kNodes = 64;

template <bool BF16>
CB_DEVICE float logit(const void* l, int64_t i) {
  if constexpr (BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(l)[i]);
  else return reinterpret_cast<const float*>(l)[i];
}

// (value, index) maximum over the block, ties to the lowest index; index -1 = none
CB_DEVICE void block_argmax(float& v, int& i, float* sv, int* si) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, nw = blockDim.x >> 5;
  auto take = [&](float ov, int oi) {
    if (oi >= 0 && (i < 0 || ov > v || (ov == v && oi < i))) { v = ov; i = oi; }
  };
  for (int o = 16; o; o >>= 1) take(__shfl_xor_sync(~0u, v, o), __shfl_xor_sync(~0u, i, o));
  __syncthreads();
  if (lane == 0) { sv[wid] = v; si[wid] = i; }
  __syncthreads();
  v = lane < nw ? sv[lane] : 0.f;
  i = lane < nw ? si[lane] : -1;
  for (int o = 16; o; o >>= 1) take(__shfl_xor_sync(~0u, v, o), __shfl_xor_sync(~0u, i, o));
}

template <bool BF16>
__global__ void __launch_bounds__(1024) tree_verify_kernel(const void* __restrict__ logits, int64_t ld, int V,
                                                           const int* __restrict__ tokens, const int* __restrict__ cu,
                                                           const int* __restrict__ parent, int N,
                                                           const float* __restrict__ uniforms,
                                                           const float* __restrict__ noise,
                                                           const float* __restrict__ temperature,
                                                           const float* __restrict__ draft, int* __restrict__ path,
                                                           int* __restrict__ n_accepted, int* __restrict__ out_tokens,
                                                           float* __restrict__ logprobs) {
  pdl_entry();
  __shared__ float red[32], red2[32];
  __shared__ int redi[32];
  __shared__ int s_tok[kNodes], s_par[kNodes];
  __shared__ float s_u[kNodes];
  const int b = blockIdx.x, t0 = cu[b], n = cu[b + 1] - t0;
  for (int i = threadIdx.x; i < N; i += blockDim.x) {
    path[b * N + i] = -1;
    out_tokens[b * N + i] = -1;
    logprobs[b * N + i] = 0.f;
    if (i < n) { s_tok[i] = tokens[t0 + i]; s_par[i] = parent[t0 + i]; s_u[i] = uniforms[t0 + i]; }
  }
  __syncthreads();
  if (n <= 0) {
    if (threadIdx.x == 0) n_accepted[b] = -1;
    return;
  }
  const float T = temperature[b];
  const bool greedy = !(T > 0.f);
  const float heat = greedy ? 1.f : T;
  float mass[kNodes];                       // of this node's rejections, in order
  int gone[kNodes];                         // their tokens
  int v = 0, steps = 0;
  while (true) {
    const char* row = reinterpret_cast<const char*>(logits) + (size_t(t0 + v) * ld) * (BF16 ? 2 : 4);
    const float* q = draft ? draft + size_t(t0 + v) * V : nullptr;
    float top = -INFINITY;
    int best = -1;
    for (int i = threadIdx.x; i < V; i += blockDim.x) {
      const float l = logit<BF16>(row, i);
      if (best < 0 || l > top) { top = l; best = i; }
    }
    block_argmax(top, best, red, redi);
    const float smax = top / heat;
    const float ref = smax == -INFINITY ? 0.f : smax;
    float e = 0.f;
    for (int i = threadIdx.x; i < V; i += blockDim.x) e += expf(logit<BF16>(row, i) / heat - ref);
    const float total = block_sum(e, red2);
    const float denom = total > 0.f ? total : (total == total ? 1.f : total);
    int k = 0;
    // remainder of token i after this node's k rejections
    auto rest = [&](int i) -> float {
      if (greedy) return i == best && total > 0.f ? 1.f : 0.f;
      float r = expf(logit<BF16>(row, i) / heat - ref) / denom;
      for (int j = 0; j < k; ++j) {
        if (q) r = fmaxf(r - q[i], 0.f) / mass[j];
        else r = gone[j] == i ? 0.f : r / mass[j];
      }
      return r;
    };
    int next = -1, x = -1;
    for (int c = v + 1; c < n && next < 0; ++c) {
      if (s_par[c] != v) continue;
      x = s_tok[c];
      if (x < 0 || x >= V) continue;        // no such token: probability zero
      const float rx = rest(x);
      if (s_u[c] * (q ? q[x] : 1.f) < rx) { next = c; break; }
      if (greedy) continue;                 // one at the maximum stays one there
      float z = 0.f;
      for (int i = threadIdx.x; i < V; i += blockDim.x) {
        const float r = rest(i);
        z += q ? fmaxf(r - q[i], 0.f) : (i == x ? 0.f : r);
      }
      z = block_sum(z, red);
      if (z > 0.f) { mass[k] = z; gone[k] = x; ++k; }
    }
    const float lse = smax + logf(total);
    if (next >= 0) {
      if (threadIdx.x == 0) {
        path[b * N + steps] = v;
        out_tokens[b * N + steps] = x;
        logprobs[b * N + steps] = logit<BF16>(row, x) / heat - lse;
      }
      ++steps;
      v = next;
      __syncthreads();
      continue;
    }
    float sc = 0.f;
    int win = -1;
    for (int i = threadIdx.x; i < V; i += blockDim.x) {
      float r = rest(i);
      if (!(r > 0.f)) continue;
      if (!greedy) r /= noise[size_t(b) * V + i];
      if (win < 0 || r > sc) { sc = r; win = i; }
    }
    __syncthreads();
    block_argmax(sc, win, red, redi);
    if (threadIdx.x == 0) {
      path[b * N + steps] = v;
      out_tokens[b * N + steps] = win;
      logprobs[b * N + steps] = win >= 0 ? logit<BF16>(row, win) / heat - lse : -INFINITY;
      n_accepted[b] = steps;
    }
    return;
  }
}

// One CTA per (cache, request); a thread owns 16 (or 4) bytes of the row and walks the path.  Node path[k] >= k and the
// path ascends, so a slot is written only after every read of it: per thread the order k = 1, 2, ... is enough.
template <typename V>
__global__ void tree_commit_kernel(const int64_t* __restrict__ caches, TreeLayout lay, int N,
                                   const int* __restrict__ path, const int* __restrict__ n_accepted) {
  pdl_entry();
  const int b = blockIdx.y;
  const int n = lay.cu[b + 1] - lay.cu[b], c = lay.ctx[b];
  const int m = min(n_accepted[b], n - 1);
  char* base = reinterpret_cast<char*>(caches[2 * blockIdx.x]);
  const int64_t bytes = caches[2 * blockIdx.x + 1];
  auto at = [&](int i) {
    const int p = c + i;
    return base + (int64_t(lay.table[size_t(b) * lay.P + p / lay.page]) * lay.page + p % lay.page) * bytes;
  };
  for (int64_t o = threadIdx.x * int64_t(sizeof(V)); o < bytes; o += blockDim.x * int64_t(sizeof(V)))
    for (int k = 1; k <= m; ++k) {
      const int i = path[b * N + k];
      if (i <= k || i >= n) continue;       // already in place, or not a node
      *reinterpret_cast<V*>(at(k) + o) = *reinterpret_cast<const V*>(at(i) + o);
    }
}

}  // namespace tree

cudaError_t tree_verify(const void* logits, bool bf16, int64_t ld, int V, const int* tokens, const int* cu,
                        const int* parent, int B, int N, const float* uniforms, const float* noise,
                        const float* temperature, const float* draft, int* path, int* n_accepted, int* out_tokens,
                        float* logprobs, cudaStream_t s) {
  if (B == 0) return cudaSuccess;
  auto f = bf16 ? tree::tree_verify_kernel<true> : tree::tree_verify_kernel<false>;
  return launch_k(f, dim3(B), 1024, 0, s, logits, ld, V, tokens, cu, parent, N, uniforms, noise, temperature, draft,
                  path, n_accepted, out_tokens, logprobs);
}

cudaError_t tree_commit(const int64_t* caches, int n, int max_row, bool wide, const TreeLayout& lay, int N, const int* path,
                        const int* n_accepted, cudaStream_t s) {
  if (n == 0 || lay.B == 0 || N < 2) return cudaSuccess;
  auto f = wide ? tree::tree_commit_kernel<uint4> : tree::tree_commit_kernel<uint32_t>;
  const int pieces = (max_row + (wide ? 15 : 3)) / (wide ? 16 : 4);
  const int threads = pieces >= 256 ? 256 : (pieces + 31) / 32 * 32;
  return launch_k(f, dim3(n, lay.B), threads, 0, s, caches, lay, N, path, n_accepted);
}

}  // namespace cb
