// Python bindings of the tree-speculation kernels.  They return the launch's CUDA error code and throw nothing: the
// arguments' checks, outputs and workspaces belong to carbon_b200/ops/spec.py, which raises Python exceptions (a C++
// exception is not safe in a build whose libstdc++ is linked statically beside torch's shared one).
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include "tree.h"

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

template <typename T>
T* ptr(const Tensor& t) { return static_cast<T*>(t.data_ptr()); }
template <typename T>
T* ptr(const OptTensor& t) { return t.has_value() && t->defined() ? ptr<T>(*t) : nullptr; }

cudaStream_t stream() { return at::cuda::getCurrentCUDAStream().stream(); }

cb::TreeLayout layout(const Tensor& cu, const Tensor& ctx, const Tensor& table, int64_t page) {
  return {ptr<int>(cu), ptr<int>(ctx), ptr<int>(table), int(table.size(0)), int(table.size(1)), int(page)};
}

int tree_mla(const Tensor& q, const Tensor& kv, const Tensor& cu, const Tensor& ctx, const Tensor& table,
             const Tensor& mask, const Tensor& req, int64_t page, double scale, const OptTensor& sink,
             const Tensor& out) {
  c10::cuda::CUDAGuard g(q.device());
  return cb::tree_mla(q.data_ptr(), q.size(0), q.size(1), q.size(2), kv.scalar_type() == at::kByte, kv.data_ptr(),
                      layout(cu, ctx, table, page), ptr<int64_t>(mask), ptr<int>(req), float(scale), ptr<float>(sink),
                      out.data_ptr(), stream());
}

// out: int32 [B (2 N + 1)] = path, tokens, n_accepted
int tree_verify(const Tensor& logits, const Tensor& tokens, const Tensor& cu, const Tensor& parent, int64_t N,
                const Tensor& uniforms, const Tensor& noise, const Tensor& temperature, const OptTensor& draft,
                const Tensor& out, const Tensor& logprobs) {
  c10::cuda::CUDAGuard g(logits.device());
  const int64_t B = cu.numel() - 1;
  int* o = ptr<int>(out);
  return cb::tree_verify(logits.data_ptr(), logits.scalar_type() == at::kBFloat16, logits.stride(0),
                         int(logits.size(1)), ptr<int>(tokens), ptr<int>(cu), ptr<int>(parent), int(B), int(N),
                         ptr<float>(uniforms), ptr<float>(noise), ptr<float>(temperature), ptr<float>(draft), o,
                         o + 2 * B * N, o + B * N, ptr<float>(logprobs), stream());
}

int tree_commit(const Tensor& caches, int64_t max_row, bool wide, const Tensor& cu, const Tensor& ctx,
                const Tensor& table, int64_t page, const Tensor& path, const Tensor& n_accepted) {
  c10::cuda::CUDAGuard g(caches.device());
  return cb::tree_commit(ptr<int64_t>(caches), int(caches.size(0)), int(max_row), wide, layout(cu, ctx, table, page),
                         int(path.size(1)), ptr<int>(path), ptr<int>(n_accepted), stream());
}

}  // namespace

void register_tree(pybind11::module_& m) {
  m.def("tree_mla", &tree_mla);
  m.def("tree_verify", &tree_verify);
  m.def("tree_commit", &tree_commit);
}
