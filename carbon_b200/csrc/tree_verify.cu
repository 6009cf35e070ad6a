// Verification of drafted token trees against the target's probabilities, and the commit of the accepted branch.
//
// Verification walks each request's tree from the root.  At node v with target probabilities p = softmax(l_v / T) the
// remainder r starts as p; child c (index order) is accepted when u_c q(x_c) < r(x_c), q the distribution its token was
// drawn from; a rejection leaves r <- max(r - q, 0) / (its sum).  Where no child is accepted the next token is
// argmax_i r_i / e_i with e ~ Exp(1) given, which is a draw from r.  Sums, maxima and probabilities are fp32.
#include "ptx.cuh"
#include "tree.h"

#include <algorithm>
#include <atomic>
#include <cfloat>

namespace cb {
namespace tree {

constexpr int kNodes = 64, kThreads = 512, kUnroll = 8, kWide = 16, kMaxCluster = 16, kShare = 1024;
constexpr float kLog2e = 1.4426950408889634f;
// Mass of a remainder, relative to the row's largest token, under which it counts as nothing left: exponentials below
// 2^-126 are flushed to zero, and a remainder above this has a token above that in any vocabulary of 2^31.
constexpr float kNothing = 0x1p-90f;

CB_DEVICE float ex2v(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Reductions over the threads of all CTAs of the cluster; every thread gets the result.  A CTA's value goes to every
// CTA's slot array through distributed shared memory; two arrays alternate, so that one exchange's slots are read
// before the next but one writes them.  WARP reduces a float4 over the first `w` lanes of a warp (w a power of two).
struct Exchange {
  float4 (*slots)[2][kMaxCluster];  // [2][2][kMaxCluster]
  float4 (*warps)[2];               // [kThreads / 32][2]
  int n, wide, rank, turn;          // wide: n or the next power of two
  // over(a, b, w): both values reduced over the first w lanes (a power of two); b only if `two`.  On entry to the last
  // reduction, lanes without a CTA hold none_a and none_b, which change nothing.
  template <typename WARP>
  CB_DEVICE void reduce(float4& a, float4& b, bool two, const float4 none_a, const float4 none_b, WARP over) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    over(a, b, 32);
    if (lane == 0) {
      warps[wid][0] = a;
      if (two) warps[wid][1] = b;
    }
    __syncthreads();
    const int t = turn++ & 1;
    if (wid == 0) {
      a = warps[lane & (kThreads / 32 - 1)][0];
      if (two) b = warps[lane & (kThreads / 32 - 1)][1];
      over(a, b, kThreads / 32);
      if (n == 1) {
        if (lane == 0) slots[t][0][0] = a;
        if (lane == 0 && two) slots[t][1][0] = b;
      } else if (lane < n) {
        auto send = [&](float4* to, const float4& v) {
          st_cluster_v4(mapa_shared(smem_u32(to), lane), __float_as_uint(v.x), __float_as_uint(v.y),
                        __float_as_uint(v.z), __float_as_uint(v.w));
        };
        send(&slots[t][0][rank], a);
        if (two) send(&slots[t][1][rank], b);
      }
    }
    if (n == 1) __syncthreads();
    else cluster_sync();
    const int at = lane & (wide - 1);
    a = at < n ? slots[t][0][at] : none_a;
    if (two) b = at < n ? slots[t][1][at] : none_b;
    if (n > 1) over(a, b, wide);
  }
  // the better of (x, i) and (ox, oi): larger value, lower index among equals (index -1: none)
  CB_DEVICE static void take(float& x, float& i, float ox, float oi) {
    const int p = __float_as_int(i), q = __float_as_int(oi);
    if (q >= 0 && (p < 0 || ox > x || (ox == x && q < p))) { x = ox; i = oi; }
  }
  // a: two rows' (maximum, sum of 2^((l - maximum) k)); b (greedy): their (maximum, its lowest index)
  CB_DEVICE void stat2(float4& a, float4& b, bool greedy, float k) {
    const float none = __int_as_float(-1);
    reduce(a, b, greedy, make_float4(-INFINITY, 0.f, -INFINITY, 0.f), make_float4(-INFINITY, none, -INFINITY, none), [&](float4& v, float4& y, int w) {
      float m = v.x, n = v.z;
      for (int o = w >> 1; o; o >>= 1) {
        m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        n = fmaxf(n, __shfl_xor_sync(~0u, n, o));
      }
      float s = v.y * ex2v((v.x - (m == -INFINITY ? 0.f : m)) * k), t = v.w * ex2v((v.z - (n == -INFINITY ? 0.f : n)) * k);
      for (int o = w >> 1; o; o >>= 1) {
        s += __shfl_xor_sync(~0u, s, o);
        t += __shfl_xor_sync(~0u, t, o);
      }
      v = make_float4(m, s, n, t);
      if (greedy) best(y, w);
    });
  }
  CB_DEVICE static void best(float4& v, int w) {
    for (int o = w >> 1; o; o >>= 1) {
      const float4 y = make_float4(__shfl_xor_sync(~0u, v.x, o), __shfl_xor_sync(~0u, v.y, o),
                                   __shfl_xor_sync(~0u, v.z, o), __shfl_xor_sync(~0u, v.w, o));
      take(v.x, v.y, y.x, y.y);
      take(v.z, v.w, y.z, y.w);
    }
  }
  // maxima of the scores .x and .z and their lowest indices .y, .w
  CB_DEVICE float4 best2(float4 a) {
    float4 unused = a;
    const float none = __int_as_float(-1);
    reduce(a, unused, false, make_float4(0.f, none, 0.f, none), a, [](float4& v, float4&, int w) { best(v, w); });
    return a;
  }
  CB_DEVICE float sum(float x) {
    float4 a = make_float4(x, 0.f, 0.f, 0.f), unused = a;
    reduce(a, unused, false, make_float4(0.f, 0.f, 0.f, 0.f), a, [](float4& v, float4&, int w) {
      for (int o = w >> 1; o; o >>= 1) v.x += __shfl_xor_sync(~0u, v.x, o);
    });
    return a.x;
  }
};

// One cluster per request: its CTAs share the vocabulary.  A visited node costs one pass over its logits (while requests
// are too few to fill HBM, or rows too short, a pass takes the node's first child along: most are accepted, and then need
// none; 20.2 -> 14.7 us for 62 chains of 18 over 688 tokens); a rejection
// of a token drawn from a distribution one pass over logits and distribution for the remainder's sum (not needed for
// the last child, whose remainder goes straight into the draw); the end one pass over logits, distribution and noise.
// A certain proposal's rejection takes its token out.  While a quarter of the row is left its mass is a difference (whose
// relative error is at most four times the sum's, about that of the exponentials).  Less may be far smaller than what
// was taken, and a child that is nearly all of what is left may be all of it, with a probability of exactly 1: then it is
// a sum, the children still in and, from one more pass over the logits (once a node), the tokens that no child has.  That
// pass at every node with a rejection took 61 trees of 16 over 20,000 tokens from 18.2 to 20.9 us, this rule to 19.0.
// What bounds it: the walk is a chain of passes, each a round of loads and one exchange (about 0.8 us), and with many
// requests the rows' bytes.  On the device, three sets of drafts each: one chain of 6 over 129,280 tokens 10.3 us, 32
// trees of 12 with distributions 45 us (about 100 MB, 2.2 TB/s: requests whose walk is short leave the device idle), 61 of
// 16 over 32,003 bf16 22.8 us.
// Asking L2 for the next rows ahead of the passes was slower (38 -> 46 us), a pass that takes the first child along is
// faster (52 -> 45 us over three sets of trees).
template <bool BF16, bool DRAFT>
__global__ void __launch_bounds__(kThreads, 2) tree_verify_kernel(
    const void* __restrict__ logits, int64_t ld, int V, const int* __restrict__ tokens, const int* __restrict__ cu,
    const int* __restrict__ parent, int N, const float* __restrict__ uniforms, const float* __restrict__ noise,
    const float* __restrict__ temperature, const float* __restrict__ draft, int clusters, int* __restrict__ path,
    int* __restrict__ n_accepted, int* __restrict__ out_tokens, float* __restrict__ logprobs) {
  pdl_entry();
  __shared__ float4 sh_slots[2][2][kMaxCluster], sh_warps[kThreads / 32][2];
  __shared__ int s_tok[kNodes], s_par[kNodes], s_child[kNodes], s_sib[kNodes], s_same[kNodes];
  // s_mass: with distributions 1 / mass of the remainder after each rejection; without, the mass of each child's later
  // siblings (every token once)
  __shared__ float s_u[kNodes], s_l[kNodes], s_q[kNodes], s_mass[kNodes];
  __shared__ float4 s_stat;                            // of the first child: maximum, sum, index of the maximum
  const int n_cta = gridDim.x / clusters;
  const int rank = n_cta == 1 ? 0 : int(cluster_ctarank()), b = blockIdx.x / n_cta;
  Exchange ex{sh_slots, sh_warps, n_cta, n_cta > 1 ? 1 << (32 - __clz(n_cta - 1)) : 1, rank, 0};
  const int t0 = cu[b], n = cu[b + 1] - t0;
  for (int i = threadIdx.x; i < N; i += kThreads) {
    if (rank == 0) {
      path[b * N + i] = -1;
      out_tokens[b * N + i] = -1;
      logprobs[b * N + i] = 0.f;
    }
    if (i < n) { s_tok[i] = tokens[t0 + i]; s_par[i] = parent[t0 + i]; s_u[i] = uniforms[t0 + i]; }
  }
  const float T = temperature[b];
  if (n_cta > 1) cluster_sync();                       // every CTA runs before any remote store
  else __syncthreads();
  if (n <= 0) {
    if (threadIdx.x == 0 && rank == 0) n_accepted[b] = -1;
    return;
  }
  if (int(threadIdx.x) < n) {   // every node's first child and next sibling (-1: none), first sibling with its token
    const int me = threadIdx.x, up = s_par[me];
    int child = -1, sib = -1, same = me;
    for (int j = n - 1; j > me; --j) {
      if (s_par[j] == me) child = j;
      if (s_par[j] == up) sib = j;
    }
    if constexpr (!DRAFT)
      for (int j = me - 1; j > 0; --j)
        if (s_par[j] == up && s_tok[j] == s_tok[me]) same = j;
    s_child[me] = child;
    s_sib[me] = sib;
    s_same[me] = same;
  }
  __syncthreads();
  const bool greedy = !(T > 0.f);
  // p = 2^((l - max) k) / total; k neither 0 (an infinite T: equal weights, and -inf stays out) nor infinite (a subnormal T)
  const float k = greedy ? kLog2e : fminf(fmaxf(kLog2e / T, __int_as_float(1)), FLT_MAX);
  const int per = (V + n_cta - 1) / n_cta, lo = rank * per, hi = min(V, lo + per);
  const float* e = noise + size_t(b) * V;
  auto row_of = [&](int node) {
    return reinterpret_cast<const char*>(logits) + (size_t(t0 + node) * ld) * (BF16 ? 2 : 4);
  };
  auto at = [](const char* row, int i) -> float {
    if constexpr (BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[i]);
    else return reinterpret_cast<const float*>(row)[i];
  };
  int v = 0, steps = 0, known = -1;                    // known: the node whose statistics are in s_stat
  while (true) {
    const char* rowp = row_of(v);
    const float* q = DRAFT ? draft + size_t(t0 + v) * V : nullptr;
    auto logit = [&](int i) { return at(rowp, i); };
    float4 st;                                         // maximum, sum, index of the maximum (greedy)
    if (v == known) {
      st = s_stat;
    } else {
      const int w = n_cta > 1 || V < 2 * kShare ? s_child[v] : -1;       // taken along
      const char* roww = w >= 0 ? row_of(w) : rowp;
      // the children's logits and draft probabilities, read while the pass runs
      if (int(threadIdx.x) < n) {
        const int up = s_par[threadIdx.x], x = s_tok[threadIdx.x];
        if (up == v || (up == w && w >= 0)) {
          const bool in = x >= 0 && x < V;
          s_l[threadIdx.x] = in ? at(row_of(up), x) : -INFINITY;
          s_q[threadIdx.x] = in ? (DRAFT ? draft[size_t(t0 + up) * V + x] : 1.f) : -1.f;   // no such token: never accepted
        }
      }
      float m[2] = {-INFINITY, -INFINITY}, s[2] = {0.f, 0.f};
      int best[2] = {-1, -1};
      auto fold = [&](int r, const float* x, int cnt, auto token) {     // token(u): x[u]'s
        float top = m[r];
        if (greedy) {
#pragma unroll
          for (int u = 0; u < kWide; ++u)
            if (u < cnt && x[u] > top) { top = x[u]; best[r] = token(u); }
        } else {
#pragma unroll
          for (int u = 0; u < kWide; ++u)
            if (u < cnt) top = fmaxf(top, x[u]);
        }
        const float ref = top == -INFINITY ? 0.f : top;
        s[r] *= ex2v((m[r] - ref) * k);
#pragma unroll
        for (int u = 0; u < kWide; ++u)
          if (u < cnt) s[r] += ex2v((x[u] - ref) * k);
        m[r] = top;
      };
      if (BF16 && per >= kThreads * 8) {
        // Eight tokens a load, on the row's own 16-byte grid (an odd length starts rows anywhere); the pieces at the ends
        // of the CTA's share are put together from single tokens.  Twice the bytes in flight: 48.6 -> 40.2 us for 83
        // chains of 11 greedy over 32,568 tokens.  Shares under a piece a thread leave threads idle and were slower
        // (25.9 -> 28.0 us at 2,700 tokens a CTA), and fp32 gains nothing from its four a load.
        auto piece = [&](const char* row, int i) -> uint4 {
          const uint16_t* h = reinterpret_cast<const uint16_t*>(row);
          if (i >= lo && i + 8 <= hi) return *reinterpret_cast<const uint4*>(h + i);
          uint32_t x[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int a = i + 2 * t;
            x[t] = (a >= lo && a < hi ? h[a] : 0xff80u) | (a + 1 >= lo && a + 1 < hi ? h[a + 1] : 0xff80u) << 16;
          }
          return make_uint4(x[0], x[1], x[2], x[3]);
        };
        auto first = [&](const char* row) {             // this thread's first piece
          const int off = int(reinterpret_cast<uintptr_t>(row + int64_t(lo) * 2) & 15) / 2;
          return lo - off + int(threadIdx.x) * 8;
        };
        auto add = [&](int r, const uint4& p, const uint4& q, int i0) {
          const uint32_t word[8] = {p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
          float x[16];
#pragma unroll
          for (int t = 0; t < 16; ++t) x[t] = __uint_as_float(t & 1 ? word[t / 2] & 0xffff0000u : word[t / 2] << 16);
          fold(r, x, 16, [&](int t) { return i0 + t + t / 8 * (kThreads - 1) * 8; });
        };
        const uint4 none = make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);      // -inf
        constexpr int STEP = kThreads * 8;
        if (w < 0) {
          for (int i0 = first(rowp); i0 < hi; i0 += 4 * STEP) {
            uint4 x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) x[u] = i0 + u * STEP < hi ? piece(rowp, i0 + u * STEP) : none;
            add(0, x[0], x[1], i0);
            add(0, x[2], x[3], i0 + 2 * STEP);
          }
        } else {
          for (int i0 = first(rowp), i1 = first(roww); i0 < hi || i1 < hi; i0 += 2 * STEP, i1 += 2 * STEP) {
            uint4 x[4];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              x[u] = i0 + u * STEP < hi ? piece(rowp, i0 + u * STEP) : none;
              x[2 + u] = i1 + u * STEP < hi ? piece(roww, i1 + u * STEP) : none;
            }
            add(0, x[0], x[1], i0);
            add(1, x[2], x[3], i1);
          }
        }
      } else if (w < 0) {                              // sixteen loads in flight
        for (int i0 = lo + int(threadIdx.x); i0 < hi; i0 += kThreads * kWide) {
          float x[kWide];
#pragma unroll
          for (int u = 0; u < kWide; ++u) x[u] = i0 + u * kThreads < hi ? logit(i0 + u * kThreads) : -INFINITY;
          fold(0, x, kWide, [&](int u) { return i0 + u * kThreads; });
        }
      } else {
        for (int i0 = lo + int(threadIdx.x); i0 < hi; i0 += kThreads * kUnroll) {
          float x[kUnroll], y[kUnroll];
#pragma unroll
          for (int u = 0; u < kUnroll; ++u) {
            const int i = i0 + u * kThreads;
            x[u] = i < hi ? logit(i) : -INFINITY;
            y[u] = i < hi ? at(roww, i) : -INFINITY;
          }
          auto token = [&](int u) { return i0 + u * kThreads; };
          fold(0, x, kUnroll, token);
          fold(1, y, kUnroll, token);
        }
      }
      float4 both = make_float4(m[0], s[0], m[1], s[1]);
      float4 idx = make_float4(m[0], __int_as_float(best[0]), m[1], __int_as_float(best[1]));
      ex.stat2(both, idx, greedy, k);
      st = make_float4(both.x, both.y, idx.y, 0.f);
      if (threadIdx.x == 0) s_stat = make_float4(both.z, both.w, idx.w, 0.f);   // read after the walk's next barrier
      known = w;
    }
    const float ref = st.x == -INFINITY ? 0.f : st.x, total = st.y;
    // a remainder's scale does not matter without distributions; NaN stays NaN
    const float inv = total != total ? total : !DRAFT ? 1.f : total > 0.f ? 1.f / total : 0.f;
    const int best = total > 0.f ? __float_as_int(st.z) : -1;
    const float lse = log2f(total);
    auto logprob = [&](float l) { return ((l - ref) * k - lse) * 0.6931471805599453f; };
    auto weight = [&](float l) { return ex2v((l - ref) * k) * inv; };
    // rejections that changed the remainder: with distributions how many, without them the last child's (0: none)
    int gone = 0;
    // the tokens of v's children up to `last` leave
    auto drop = [&](float* r, int i0, int last) {
      for (int c = s_child[v]; c >= 0 && c <= last; c = s_sib[c]) {
        const int x = s_tok[c];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (x == i0 + u * kThreads) r[u] = 0.f;
      }
    };
    // remainder of the tokens i0, i0 + kThreads, ... with logits r[] after them
    auto rest = [&](float* r, const float* qi, int i0, int cnt) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (u < cnt) r[u] = weight(r[u]);
      if constexpr (DRAFT) {
        for (int j = 0; j < gone; ++j) {
          const float f = s_mass[j];
#pragma unroll
          for (int u = 0; u < kUnroll; ++u)
            if (u < cnt) r[u] = fmaxf(r[u] - qi[u], 0.f) * f;
        }
      } else {
        drop(r, i0, gone);
      }
    };
    int next = -1, x = -1;
    float mass = total;                                // without distributions: of the remainder
    float others = -1.f;                               // and of the tokens that are no child's, once summed
    bool open = false;                                 // the last child's rejection goes into the draw
    auto sum_others = [&]() -> float {
      if (int(threadIdx.x) < n && s_par[threadIdx.x] == v) {
        float later = 0.f;
        for (int d = s_sib[threadIdx.x]; d >= 0; d = s_sib[d])
          if (s_same[d] == d) later += weight(s_l[d]);
        s_mass[threadIdx.x] = later;
      }
      float z = 0.f;
      for (int i0 = lo + int(threadIdx.x); i0 < hi; i0 += kThreads * kUnroll) {
        float r[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) r[u] = i0 + u * kThreads < hi ? logit(i0 + u * kThreads) : -INFINITY;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) r[u] = weight(r[u]);
        drop(r, i0, n);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) z += r[u];
      }
      return ex.sum(z);                                // its barrier publishes s_mass
    };
    for (int c = s_child[v]; c >= 0; c = s_sib[c]) {
      x = s_tok[c];
      const float qx = s_q[c];
      if (qx < 0.f) continue;                          // no such token
      float rx = s_l[c];
      if (greedy) rx = x == best ? 1.f : 0.f;
      else if constexpr (DRAFT) rest(&rx, &qx, x, 1);
      else rx = s_same[c] <= gone ? 0.f : weight(rx);
      if (!DRAFT && !greedy && gone && others < 0.f && rx > 0.999f * mass) {
        others = sum_others();
        mass = others + s_mass[gone];
      }
      if (s_u[c] * (DRAFT || greedy ? qx : mass) < rx) { next = c; break; }
      if (greedy) continue;                            // one at the maximum stays one there
      if (!DRAFT && !(rx > 0.f)) continue;             // a token that has left, or was never there
      if (s_sib[c] < 0) {
        open = true;
        break;
      }
      float z = 0.f;
      if constexpr (!DRAFT) {
        if (others < 0.f && mass - rx >= 0.25f * total) {
          mass -= rx;
          gone = c;
          continue;
        }
        if (others < 0.f) others = sum_others();
        if (others + s_mass[c] > kNothing) { mass = others + s_mass[c]; gone = c; }    // else the remainder stays
      } else {
        for (int i0 = lo + int(threadIdx.x); i0 < hi; i0 += kThreads * kUnroll) {
          float r[kUnroll], qi[kUnroll];
#pragma unroll
          for (int u = 0; u < kUnroll; ++u) {
            const int i = i0 + u * kThreads;
            r[u] = i < hi ? logit(i) : -INFINITY;
            qi[u] = i < hi ? q[i] : 0.f;
          }
          rest(r, qi, i0, kUnroll);
#pragma unroll
          for (int u = 0; u < kUnroll; ++u) z += fmaxf(r[u] - qi[u], 0.f);
        }
        z = ex.sum(z);
        if (z > 0.f) {
          if (threadIdx.x == 0) s_mass[gone] = 1.f / z;
          __syncthreads();
          ++gone;
        }
      }
    }
    if (next >= 0) {
      if (threadIdx.x == 0 && rank == 0) {
        path[b * N + steps] = v;
        out_tokens[b * N + steps] = x;
        logprobs[b * N + steps] = logprob(s_l[next]);
      }
      ++steps;
      v = next;
      __syncthreads();                                 // s_l, s_q, s_mass are rewritten
      continue;
    }
    int win = best;
    if (!greedy) {
      // The draw: r / e is compared as r * e' > r' * e.  Second result: the draw from the remainder before the last
      // rejection, which stands if that left nothing.
      float r1 = 0.f, e1 = 1.f, r0 = 0.f, e0 = 1.f;
      int w1 = -1, w0 = -1;
      const bool with_q = DRAFT && (open || gone > 0);  // else the distribution is not read
      for (int i0 = lo + int(threadIdx.x); i0 < hi; i0 += kThreads * kUnroll) {
        float r[kUnroll], qi[kUnroll], ei[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const int i = i0 + u * kThreads;
          r[u] = i < hi ? logit(i) : -INFINITY;
          qi[u] = with_q && i < hi ? q[i] : 0.f;
          ei[u] = i < hi ? e[i] : 1.f;
        }
        rest(r, qi, i0, kUnroll);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const int i = i0 + u * kThreads;
          const float d = !open ? r[u] : DRAFT ? fmaxf(r[u] - qi[u], 0.f) : i == x ? 0.f : r[u];
          if (d * e1 > r1 * ei[u]) { r1 = d; e1 = ei[u]; w1 = i; }
          if (DRAFT && open && r[u] * e0 > r0 * ei[u]) { r0 = r[u]; e0 = ei[u]; w0 = i; }
        }
      }
      const float4 w = ex.best2(make_float4(r1 / e1, __int_as_float(w1), r0 / e0, __int_as_float(w0)));
      win = __float_as_int(w.y);
      if (DRAFT && win < 0) win = __float_as_int(w.w);
      if (!DRAFT && open && win < 0) win = x;          // nothing else was left
    }
    if (threadIdx.x == 0 && rank == 0) {
      path[b * N + steps] = v;
      out_tokens[b * N + steps] = win;
      logprobs[b * N + steps] = win >= 0 ? logprob(logit(win)) : -INFINITY;
      n_accepted[b] = steps;
    }
    return;
  }
}

// One CTA per (cache, request); a thread owns 16 (or 4) bytes of the row and walks the path, eight rows in flight.  Node
// path[k] >= k and the path ascends, so a slot is written only after every read of it: per thread the order of k is
// enough, and reading a later row early is harmless.  The rows' slots are looked up once per CTA, in parallel: a lookup
// per row made 32 requests x 61 layers 7.7 us, now 4.8 us (19 MB moved; latency of one dependent chain, launch included).
template <typename V>
__global__ void __launch_bounds__(256) tree_commit_kernel(const int64_t* __restrict__ caches, TreeLayout lay, int N,
                                                          const int* __restrict__ path,
                                                          const int* __restrict__ n_accepted) {
  __shared__ int s_from[kNodes], s_to[kNodes];
  __shared__ int s_moves;
  const int b = blockIdx.y;
  const int n = lay.cu[b + 1] - lay.cu[b], c = lay.ctx[b];               // made by the host
  char* base = reinterpret_cast<char*>(caches[2 * blockIdx.x]);
  const int64_t bytes = caches[2 * blockIdx.x + 1];
  pdl_entry();
  const int m = min(n_accepted[b], n - 1);
  if (m <= 0) return;
  if (threadIdx.x < 32) {
    auto slot = [&](int i) {
      const int p = c + i;
      return lay.table[size_t(b) * lay.P + p / lay.page] * lay.page + p % lay.page;
    };
    int moves = 0;
    for (int k0 = 1; k0 <= m; k0 += 32) {
      const int k = k0 + int(threadIdx.x);
      const int i = k <= m ? path[b * N + k] : -1;
      const bool move = i > k && i < n;                // else already in place, or not a node
      const uint32_t all = __ballot_sync(~0u, move);
      if (move) {
        const int at = moves + __popc(all & ((1u << threadIdx.x) - 1));
        s_from[at] = slot(i);
        s_to[at] = slot(k);
      }
      moves += __popc(all);
    }
    if (threadIdx.x == 0) s_moves = moves;
  }
  __syncthreads();
  const int moves = s_moves;
  for (int64_t o = threadIdx.x * int64_t(sizeof(V)); o < bytes; o += blockDim.x * int64_t(sizeof(V)))
    for (int k0 = 0; k0 < moves; k0 += 8) {
      V v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k0 + k < moves) v[k] = *reinterpret_cast<const V*>(base + s_from[k0 + k] * bytes + o);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k0 + k < moves) *reinterpret_cast<V*>(base + s_to[k0 + k] * bytes + o) = v[k];
    }
}

// Clusters of c CTAs that the device holds at once: a property of device and kernel, asked once.
template <typename F>
cudaError_t clusters_that_fit(F f, int variant, int c, int* fit) {
  constexpr int kDevices = 16;
  static std::atomic<int> known[kDevices][4][kMaxCluster + 1];           // 1 + clusters
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < kDevices && (*fit = known[dev][variant][c].load() - 1) >= 0) return cudaSuccess;
  if (c > 8 && (e = cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess) return e;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = c; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(c);
  cfg.blockDim = dim3(kThreads);
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if ((e = cudaOccupancyMaxActiveClusters(fit, f, &cfg)) != cudaSuccess) return e;
  if (dev < kDevices) known[dev][variant][c].store(*fit + 1);
  return cudaSuccess;
}

}  // namespace tree

cudaError_t tree_verify(const void* logits, bool bf16, int64_t ld, int V, const int* tokens, const int* cu,
                        const int* parent, int B, int N, const float* uniforms, const float* noise,
                        const float* temperature, const float* draft, int* path, int* n_accepted, int* out_tokens,
                        float* logprobs, cudaStream_t s) {
  if (B == 0) return cudaSuccess;
  auto f = bf16 ? (draft ? tree::tree_verify_kernel<true, true> : tree::tree_verify_kernel<true, false>)
                : (draft ? tree::tree_verify_kernel<false, true> : tree::tree_verify_kernel<false, false>);
  // CTAs per request: as many as keep all requests on the device at once (two CTAs per SM, a cluster within one GPC),
  // each with kShare tokens or more.  16 chains over 129,280 tokens take 20.9 us with 16 CTAs each, which do not all
  // fit, 18.0 with 13; 86 over 10,260 tokens 13.7 with 2, 12.5 with 3.
  int c = std::max(1, std::min(tree::kMaxCluster, V / tree::kShare));
  cudaError_t e = cudaSuccess;
  while (c > 1) {
    int fit = 0;
    if ((e = tree::clusters_that_fit(f, (bf16 ? 2 : 0) + (draft ? 1 : 0), c, &fit)) != cudaSuccess) return e;
    if (B <= fit) break;
    --c;
  }
  if (c > 8 && (e = cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess) return e;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = c; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(B) * c);
  cfg.blockDim = dim3(tree::kThreads);
  cfg.stream = s;
  cfg.attrs = pdl_enabled() ? attr : attr + 1;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, f, logits, ld, V, tokens, cu, parent, N, uniforms, noise, temperature, draft, B,
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
