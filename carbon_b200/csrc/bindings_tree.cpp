// Python bindings of the tree-speculation kernels.  They return the launch's CUDA error code and throw nothing: the
// arguments' checks, outputs and workspaces belong to carbon_b200/ops/spec.py, which raises Python exceptions (a C++
// exception is not safe in a build whose libstdc++ is linked statically beside torch's shared one).
#include <torch/extension.h>
#include <torch/cuda.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <algorithm>
#include <cstring>
#include <queue>
#include <tuple>
#include <vector>
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

// Split of one attention call over `clusters` CTA pairs (csrc/tree.h: TreeWork).  Every row tile of every request is a
// list of ceil((ctx + n) / 128) key tiles; longest first, each goes to the pair with the least work so far.  Where it
// would pass a share of the work it is cut there and the rest goes on to the next pair (partial results are merged).
// Several shares from the even one up are tried, and the one with the least cost is taken: the longest pair's tiles plus
// kOver for every item's start and end, and the merge (kMerge at all, kPart per partial result: 256 KB written and
// read).  64 requests of 1250 to 2500 keys, one row tile each: 53 us (67 us at the even share alone).
// The row tiles of a request are handed out one after the other, so they run at about the same time and read its keys
// from L2.
// -> int32 tensor (16-byte aligned parts): first [clusters + 1], items [*, 8], merges [*, 6], whole key tiles (request,
// tile) [*, 2], first of them per request [B]; and the counts of CTA pairs, items, merges, partial results, whole key
// tiles, key tiles over all items and the most partial results of a row tile
std::tuple<Tensor, std::vector<int64_t>> tree_schedule(const std::vector<int64_t>& n, const std::vector<int64_t>& ctx,
                                                       int64_t H, int64_t clusters) {
  constexpr int64_t kTile = 128, kOver = 2;
  constexpr double kMerge = 1.5, kPart = 0.04;
  const int64_t B = int64_t(n.size());
  std::vector<int64_t> cu(B + 1, 0);
  for (int64_t b = 0; b < B; ++b) cu[b + 1] = cu[b] + n[b];
  struct Row { int64_t b, row, tiles; };
  std::vector<Row> rows;
  int64_t total = 0;
  for (int64_t b = 0; b < B; ++b) {
    const int64_t tiles = (ctx[b] + n[b] + kTile - 1) / kTile;
    for (int64_t r = 0; r < (n[b] * H + 127) / 128; ++r, total += tiles + kOver) rows.push_back({b, r, tiles});
  }
  std::stable_sort(rows.begin(), rows.end(), [](const Row& x, const Row& y) { return x.tiles > y.tiles; });
  clusters = std::max<int64_t>(1, clusters);
  using Load = std::pair<int64_t, int64_t>;                       // (work, pair)
  std::vector<std::vector<cb::TreeItem>> lists;
  std::vector<cb::TreeMerge> merges;
  int64_t parts = 0;
  auto assign = [&](int64_t share, bool force) -> bool {
    std::priority_queue<Load, std::vector<Load>, std::greater<Load>> heap;
    for (int64_t c = 0; c < clusters; ++c) heap.push({0, c});
    lists.assign(clusters, {});
    merges.clear();
    parts = 0;
    for (const Row& r : rows) {
      const int64_t first_part = parts;
      std::vector<std::pair<int64_t, size_t>> pieces;
      for (int64_t at = 0; at < r.tiles;) {
        const Load ld = heap.top();
        heap.pop();
        const int64_t rest = r.tiles - at, room = share - ld.first - kOver;
        if (!force && room < 1) return false;
        const int64_t take = force ? rest : std::min(rest, room);    // a remainder of one tile goes on, too
        auto& list = lists[ld.second];
        pieces.push_back({ld.second, list.size()});
        list.push_back({int(r.b), int(r.row), int(at), int(take), -1, int(ctx[r.b]), int(cu[r.b]), int(n[r.b])});
        heap.push({ld.first + take + kOver, ld.second});
        at += take;
      }
      if (pieces.size() > 1) {
        for (auto& [c, i] : pieces) lists[c][i].part = int(parts++);
        merges.push_back({int(r.row), int(first_part), int(pieces.size()), int(cu[r.b]), int(n[r.b] * H), 0});
      }
    }
    return true;
  };
  const int64_t even = std::max((total + clusters - 1) / clusters, 1 + kOver);
  double least = 0;
  int64_t take = -1;
  for (int64_t share = even, tries = 0; tries < 16; ++tries, share += std::max<int64_t>(1, even / 24)) {
    if (!assign(share, false)) continue;
    int64_t longest = 0;
    for (const auto& l : lists) {
      int64_t w = 0;
      for (const auto& it : l) w += it.n_tiles + kOver;
      longest = std::max(longest, w);
    }
    const double cost = double(longest) + (parts ? kMerge + kPart * double(parts) : 0.0);
    if (take < 0 || cost < least) { least = cost; take = share; }
    if (!parts) break;                                            // a larger share changes nothing any more
  }
  assign(std::max(take, even), take < 0);
  int64_t used = 0, n_items = 0;
  for (auto& l : lists) { used += !l.empty(); n_items += int64_t(l.size()); }
  std::stable_sort(lists.begin(), lists.end(), [](const auto& x, const auto& y) { return !x.empty() && y.empty(); });
  const int64_t head = (used + 1 + 3) / 4 * 4;
  int64_t n_stage = 0, work = 0;
  for (int64_t b = 0; b < B; ++b) n_stage += n[b] ? ctx[b] / kTile : 0;
  for (const Row& r : rows) work += r.tiles;
  const int64_t tail = head + n_items * 8 + int64_t(merges.size()) * 6;
  auto out = torch::empty({(tail + 2 * n_stage + B + 3) / 4 * 4}, torch::kInt32);
  int* o = ptr<int>(out);
  int at = 0;
  for (int64_t c = 0; c < head; ++c) {
    o[c] = at;
    if (c < used)
      for (const auto& it : lists[c]) std::memcpy(o + head + 8 * at++, &it, sizeof it);
  }
  if (!merges.empty()) std::memcpy(o + head + 8 * n_items, merges.data(), merges.size() * sizeof merges[0]);
  int* st = o + tail;
  int* first = st + 2 * n_stage;
  int k = 0;
  for (int64_t b = 0; b < B; ++b) {
    first[b] = k;
    for (int64_t t = 0; n[b] && t < ctx[b] / kTile; ++t, ++k) {
      st[2 * k] = int(b);
      st[2 * k + 1] = int(t);
    }
  }
  int64_t most = 0;
  for (const auto& m : merges) most = std::max<int64_t>(most, m.n);
  return {out, {used, n_items, int64_t(merges.size()), parts, n_stage, work, most}};
}

// The lists of a TreePlan with the default masks (each node's ancestors and itself), in one pinned int32 buffer:
// work (tree_schedule) | masks [T, 2] | cu [B + 1] | ctx [B] | req [T] | parent [T] | pos [T] | slot [T] | table [B, P] |
// status (0).  Returns (0, buffer, counts, [work length, T, N, P, largest page]), or (-1, ...) where an argument does not
// fit: the caller's own checks then say which.
std::tuple<int, Tensor, std::vector<int64_t>, std::vector<int64_t>> tree_plan(
    const std::vector<std::vector<int64_t>>& tables, const std::vector<int64_t>& ctx,
    const std::vector<std::vector<int64_t>>& parents, int64_t page, int64_t H, int64_t clusters) {
  const int64_t B = int64_t(parents.size());
  const auto refuse = std::make_tuple(-1, Tensor(), std::vector<int64_t>(), std::vector<int64_t>());
  if (int64_t(tables.size()) != B || int64_t(ctx.size()) != B || page < 1 || H < 1) return refuse;
  std::vector<int64_t> n(B);
  int64_t T = 0, N = 0, P = 1, top = -1;
  for (int64_t b = 0; b < B; ++b) {
    const int64_t k = n[b] = int64_t(parents[b].size()), have = int64_t(tables[b].size());
    if (k > 64 || ctx[b] < 0 || (ctx[b] + k + page - 1) / page > have) return refuse;
    for (int64_t i = 0; i < k; ++i)
      if (i ? parents[b][i] < 0 || parents[b][i] >= i : parents[b][i] != -1) return refuse;
    for (int64_t pg : tables[b]) {
      if (pg < 0 || (pg + 1) * page > (int64_t(1) << 31) - 1) return refuse;
      top = std::max(top, pg);
    }
    T += k;
    N = std::max(N, k);
    P = std::max(P, have);
  }
  Tensor work = torch::empty({0}, torch::kInt32);
  std::vector<int64_t> counts;
  if (T) std::tie(work, counts) = tree_schedule(n, ctx, H, clusters);
  const int64_t W = work.numel();
  auto out = torch::empty({W + 2 * T + B + 1 + B + 4 * T + B * P + 1},
                          torch::TensorOptions().dtype(torch::kInt32).pinned_memory(torch::cuda::is_available()));
  int* o = ptr<int>(out);
  if (W) std::memcpy(o, ptr<int>(work), W * sizeof(int));
  int* masks = o + W;
  int* cu = masks + 2 * T;
  int* cx = cu + B + 1;
  int *req = cx + B, *par = req + T, *pos = par + T, *slot = pos + T, *table = slot + T;
  int64_t t = 0;
  cu[0] = 0;
  for (int64_t b = 0; b < B; ++b) {
    uint64_t mask[64];
    int depth[64];
    for (int64_t i = 0; i < n[b]; ++i, ++t) {
      const int64_t up = parents[b][i], at = ctx[b] + i;
      mask[i] = (uint64_t(1) << i) | (i ? mask[up] : 0);
      depth[i] = i ? depth[up] + 1 : 0;
      std::memcpy(masks + 2 * t, &mask[i], 8);
      req[t] = int(b);
      par[t] = int(up);
      pos[t] = int(ctx[b] + depth[i]);
      slot[t] = int(tables[b][at / page] * page + at % page);
    }
    cu[b + 1] = int(t);
    cx[b] = int(ctx[b]);
    for (int64_t i = 0; i < P; ++i) table[b * P + i] = i < int64_t(tables[b].size()) ? int(tables[b][i]) : 0;
  }
  table[B * P] = 0;
  return {0, out, counts, {W, T, N, P, top}};
}

// work: tree_schedule's tensor on the device, counts its counts; buf: workspace of the partial outputs, then (m, l);
// staged: workspace of the dense key rows, if they are to be staged
int tree_mla(const Tensor& q, const Tensor& kv, const Tensor& cu, const Tensor& ctx, const Tensor& table,
             const Tensor& mask, int64_t page, const Tensor& work, const std::vector<int64_t>& counts,
             const OptTensor& buf, const OptTensor& staged, double scale, const OptTensor& sink, const Tensor& status,
             const Tensor& out) {
  c10::cuda::CUDAGuard g(q.device());
  const int* w = ptr<int>(work);
  const int64_t head = (counts[0] + 1 + 3) / 4 * 4;
  cb::TreeWork tw;
  tw.first = w;
  tw.items = reinterpret_cast<const cb::TreeItem*>(w + head);
  tw.merges = reinterpret_cast<const cb::TreeMerge*>(w + head + 8 * counts[1]);
  tw.clusters = int(counts[0]);
  tw.n_merges = int(counts[2]);
  tw.most_parts = int(counts[6]);
  const int* st = w + head + 8 * counts[1] + 6 * counts[2];
  tw.stage = reinterpret_cast<const int2*>(st);
  tw.stage_at = st + 2 * counts[4];
  tw.n_stage = int(counts[4]);
  float* part = ptr<float>(buf);
  return cb::tree_mla(q.data_ptr(), q.size(0), q.size(1), q.size(2), kv.scalar_type() == at::kByte, kv.data_ptr(),
                      kv.size(0), layout(cu, ctx, table, page), tw, ptr<int64_t>(mask), float(scale), ptr<float>(sink),
                      part, part ? part + counts[3] * 128 * 512 : nullptr, ptr<void>(staged), ptr<int>(status), out.data_ptr(), stream());
}

// Whether t is a contiguous tensor of this type, size and device.
bool fits(const Tensor& t, at::ScalarType dt, const c10::Device& dev, std::initializer_list<int64_t> shape) {
  return t.scalar_type() == dt && t.device() == dev && t.is_contiguous() && t.sizes().equals(shape);
}

// out: int32 [B (3 N + 1)] = path [B, N], n_accepted [B], tokens [B, N], logprobs [B, N] (fp32), returned as views.
// Code -1: an argument does not fit (the caller says which).
std::tuple<int, Tensor, Tensor, Tensor, Tensor> tree_verify(const Tensor& logits, const Tensor& tokens,
                                                            const Tensor& cu, const Tensor& parent, int64_t N,
                                                            const Tensor& uniforms, const Tensor& noise,
                                                            const Tensor& temperature, const OptTensor& draft,
                                                            const Tensor& out) {
  const c10::Device dev = cu.device();
  const int64_t B = cu.numel() - 1, T = parent.numel();
  const bool bf16 = logits.scalar_type() == at::kBFloat16;
  bool ok = logits.dim() == 2 && logits.size(0) == T && (bf16 || logits.scalar_type() == at::kFloat) &&
            logits.device() == dev;
  const int64_t V = ok ? logits.size(1) : 0;
  ok = ok && V > 0 && V < (int64_t(1) << 31) && (T == 0 || logits.stride(1) == 1) &&
       fits(tokens, at::kInt, dev, {T}) && fits(uniforms, at::kFloat, dev, {T}) &&
       fits(noise, at::kFloat, dev, {B, V}) && fits(temperature, at::kFloat, dev, {B}) &&
       (!draft.has_value() || fits(*draft, at::kFloat, dev, {T, V}));
  if (!ok) return {-1, out, out, out, out};
  c10::cuda::CUDAGuard g(dev);
  int* o = ptr<int>(out);
  const int e = cb::tree_verify(logits.data_ptr(), bf16, logits.stride(0), int(V), ptr<int>(tokens), ptr<int>(cu),
                                ptr<int>(parent), int(B), int(N), ptr<float>(uniforms), ptr<float>(noise),
                                ptr<float>(temperature), ptr<float>(draft), o, o + B * N, o + B * (N + 1),
                                reinterpret_cast<float*>(o + B * (2 * N + 1)), stream());
  at::AutoDispatchBelowADInplaceOrView plain;           // views of a fresh tensor: nothing for autograd to note
  return {e, out.as_strided({B, N}, {N, 1}, 0), out.as_strided({B}, {1}, B * N),
          out.as_strided({B, N}, {N, 1}, B * (N + 1)), out.view(at::kFloat).as_strided({B, N}, {N, 1}, B * (2 * N + 1))};
}

int tree_commit(const Tensor& caches, int64_t max_row, bool wide, const Tensor& cu, const Tensor& ctx,
                const Tensor& table, int64_t page, const Tensor& path, const Tensor& n_accepted) {
  c10::cuda::CUDAGuard g(caches.device());
  return cb::tree_commit(ptr<int64_t>(caches), int(caches.size(0)), int(max_row), wide, layout(cu, ctx, table, page),
                         int(path.size(1)), ptr<int>(path), ptr<int>(n_accepted), stream());
}

}  // namespace

void register_tree(pybind11::module_& m) {
  m.def("tree_plan", &tree_plan);
  m.def("tree_mla_clusters", [] { return cb::tree_mla_clusters(); });
  m.def("tree_mla", &tree_mla);
  m.def("tree_verify", &tree_verify);
  m.def("tree_commit", &tree_commit);
}
