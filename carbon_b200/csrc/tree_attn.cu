// Attention of drafted token trees over the paged latent cache.
//
//   o[t, h, :] = sum_j w_j kv_j[:512] / (sum_j w_j + exp(sink_h)),   w_j = exp(scale * q[t, h] . kv_j)
//
// over the keys j that node t of request b sees: every position before ctx[b], and position ctx[b] + i for each bit i
// of mask[t].  One warp per (node, head): a lane holds 16 of the 512 latent dims and 2 of the RoPE dims, the running
// maximum and sum are kept in fp32.
#include <cuda_fp16.h>
#include "common.cuh"
#include "tree.h"

namespace cb {
namespace tree {

template <bool F8>
__global__ void __launch_bounds__(256) tree_mla_warp_kernel(const void* __restrict__ qv, const void* __restrict__ kvv,
                                                            TreeLayout lay, const int64_t* __restrict__ mask,
                                                            const int* __restrict__ req, int T, int H, int D,
                                                            float scale_log2, const float* __restrict__ sink,
                                                            __nv_bfloat16* __restrict__ out) {
  pdl_entry();
  const int w = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, lane = threadIdx.x & 31;
  if (w >= T * H) return;
  const int t = w / H, h = w % H, b = req[t];
  const int c = lay.ctx[b], n = lay.cu[b + 1] - lay.cu[b];
  const uint64_t m = uint64_t(mask[t]);
  const int row_bytes = F8 ? (D == 576 ? 656 : 528) : D * 2;
  const size_t qo = (size_t(t) * H + h) * D;
  float q[18];
  if constexpr (F8) {
    const __half* p = reinterpret_cast<const __half*>(qv) + qo;
    for (int i = 0; i < 16; ++i) q[i] = __half2float(p[lane * 16 + i]);
    for (int i = 0; i < 2; ++i) q[16 + i] = D == 576 ? __half2float(p[512 + lane * 2 + i]) : 0.f;
  } else {
    const __nv_bfloat16* p = reinterpret_cast<const __nv_bfloat16*>(qv) + qo;
    for (int i = 0; i < 16; ++i) q[i] = __bfloat162float(p[lane * 16 + i]);
    for (int i = 0; i < 2; ++i) q[16 + i] = D == 576 ? __bfloat162float(p[512 + lane * 2 + i]) : 0.f;
  }
  float top = -INFINITY, total = 0.f, acc[16];
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
  for (int j = 0; j < c + n; ++j) {
    if (j >= c && !((m >> (j - c)) & 1)) continue;
    const int slot = lay.table[size_t(b) * lay.P + j / lay.page] * lay.page + j % lay.page;
    const uint8_t* r = reinterpret_cast<const uint8_t*>(kvv) + size_t(slot) * row_bytes;
    float k[18];
    if constexpr (F8) {
      const uint4 v = *reinterpret_cast<const uint4*>(r + lane * 16 + (lane >= 16 ? 16 : 0));
      const float sc = ue8m0_to_float(r[256 + (lane >> 2)]);
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
      for (int i = 0; i < 16; ++i) {
        __nv_fp8_e4m3 e;
        e.__x = (u[i >> 2] >> (8 * (i & 3))) & 0xff;
        k[i] = float(e) * sc;
      }
      for (int i = 0; i < 2; ++i)
        k[16 + i] = D == 576 ? __half2float(reinterpret_cast<const __half*>(r + 528)[lane * 2 + i]) : 0.f;
    } else {
      const __nv_bfloat16* p = reinterpret_cast<const __nv_bfloat16*>(r);
      for (int i = 0; i < 16; ++i) k[i] = __bfloat162float(p[lane * 16 + i]);
      for (int i = 0; i < 2; ++i) k[16 + i] = D == 576 ? __bfloat162float(p[512 + lane * 2 + i]) : 0.f;
    }
    float s = 0.f;
    for (int i = 0; i < 18; ++i) s += q[i] * k[i];
    s = warp_sum(s) * scale_log2;
    const float nt = fmaxf(top, s);
    const float ref = nt == -INFINITY ? 0.f : nt;
    const float keep = exp2f(top - ref), e = exp2f(s - ref);
    total = total * keep + e;
    for (int i = 0; i < 16; ++i) acc[i] = acc[i] * keep + e * k[i];
    top = nt;
  }
  if (sink) total += exp2f(sink[h] * 1.4426950408889634f - (top == -INFINITY ? 0.f : top));
  const float inv = total > 0.f ? 1.f / total : (total == total ? 0.f : total);   // NaN scores stay visible
  __nv_bfloat16* o = out + (size_t(t) * H + h) * 512 + lane * 16;
  for (int i = 0; i < 16; ++i) o[i] = __float2bfloat16(acc[i] * inv);
}

}  // namespace tree

cudaError_t tree_mla(const void* q, int T, int H, int D, bool f8, const void* kv, const TreeLayout& lay,
                     const int64_t* mask, const int* req, float scale, const float* sink, void* out, cudaStream_t s) {
  if (T == 0) return cudaSuccess;
  const dim3 grid((int64_t(T) * H + 7) / 8);
  auto* o = reinterpret_cast<__nv_bfloat16*>(out);
  const float sl = scale * 1.4426950408889634f;
  return f8 ? launch_k(tree::tree_mla_warp_kernel<true>, grid, 256, 0, s, q, kv, lay, mask, req, T, H, D, sl, sink, o)
            : launch_k(tree::tree_mla_warp_kernel<false>, grid, 256, 0, s, q, kv, lay, mask, req, T, H, D, sl, sink, o);
}

}  // namespace cb
