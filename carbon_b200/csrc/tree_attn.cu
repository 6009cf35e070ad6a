// Attention of drafted token trees over the paged latent cache, on tcgen05 (sm_100a).
//
//   o[t, h, :] = sum_j w_j kv_j[:512] / (sum_j w_j + exp(sink_h)),   w_j = exp(scale * q[t, h] . kv_j)
//
// over the keys j that node t of request b sees: every position before ctx[b], and position ctx[b] + i for each bit i
// of mask[t].  All heads of all nodes of a request share its key rows, so the nodes x heads rows are cut into 128-row
// tiles and a CTA pair (cta_group::2, M = 128) runs one of them: each CTA holds 64 rows, its O [64 x 512] fills 256
// TMEM columns (an M = 128 pair tile keeps the first half of N in lanes 0-63 and the second half in lanes 64-127),
// which leaves room for two score tiles.  (One CTA with M = 128 rows would need all 512 columns for O.)
//
// Three launches: tree_stage_kernel brings the key rows that the tensor core cannot take as they lie in the cache (fp8
// rows, rows of small pages, and always the last tiles, whose rows end or belong to the tree) into a dense buffer;
// tree_mla_kernel does the attention; tree_merge_kernel joins row tiles whose keys were split over CTA pairs.
#include <cudaTypedefs.h>
#include <cuda_fp16.h>
#include "ptx.cuh"
#include "tree.h"

namespace cb {
namespace tree {

constexpr int KT = 128;                    // keys per tile: N of Q·K^T (64 from each CTA), K of P·V
constexpr int CH = 64 * 128;               // chunk: 64 rows x 64 dims of 16-bit values, 128-byte swizzled
constexpr int SLOTS = 9;                   // chunks of a stage: the CTA's 64 keys, 576 dims
constexpr int STAGE = SLOTS * CH;
constexpr int NST = 2;
constexpr int TM_O = 0, TM_S = 256;        // TMEM columns: O 256, two score buffers of 64
constexpr int SM_WARPS = 8;                // softmax warps: two per 32 TMEM lanes, each one half of the score columns
constexpr int THREADS = 128 + SM_WARPS * 32;
constexpr int SMEM_USED = SLOTS * CH + NST * STAGE + CH + 2048 + 256;
constexpr int SMEM = SMEM_USED + 768;      // 227 KB; the base is 256-byte aligned at least (checked by the kernel)
constexpr float kRescale = 8.f;            // O is rescaled when the running maximum grows by more than 2^8

struct Params {
  TreeLayout lay;
  TreeWork work;
  const int64_t* mask;
  const int* bad;
  int H, stage_all, box;                   // box: cache rows one TMA load takes (page-contiguous)
  float scale_log2;
  const float* sink;
  float* part_o;
  float* part_ml;
  int* status;
  __nv_bfloat16* out;
};

CB_DEVICE uint64_t desc_mn(const void* p) {  // MN-major operand: 64-dim chunks CH apart, 8-key groups 1024 B apart
  const uint64_t addr = smem_u32(p);
  return ((addr >> 4) & 0x3FFFull) | (uint64_t(CH >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
         (uint64_t(2) << 61);
}
CB_DEVICE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
CB_DEVICE uint32_t pack2(float a, float b, bool f16) {
  if (f16) {
    __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  return pack_bf16x2(a, b);
}
CB_DEVICE void softmax_sync() { asm volatile("bar.sync 1, %0;" ::"n"(SM_WARPS * 32) : "memory"); }

// ---------------------------------------------------------------------------------------------------------------
// Rows [tile * 128, ...) of a request -> block of the staging buffer, zeros past its last node.  fp8 rows are expanded
// to fp16 (exact).  A tree row with a NaN or an infinity is staged as zeros and marked in bad[]: nodes of other
// branches multiply it by a weight of zero, nodes that see it are made NaN by the attention kernel.  One warp per row.
// ---------------------------------------------------------------------------------------------------------------
CB_DEVICE bool nonfinite16(uint32_t v, uint32_t expo) {      // either half has all exponent bits set
  return (v & expo) == expo || ((v >> 16) & expo) == expo;
}

template <bool F8>
__global__ void __launch_bounds__(256) tree_stage_kernel(const uint8_t* __restrict__ kv, TreeLayout lay,
                                                         const int2* __restrict__ blocks, int D,
                                                         uint16_t* __restrict__ staged, int* __restrict__ bad) {
  pdl_entry();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int2 blk = blocks[blockIdx.x >> 2];
  const int b = blk.x, c = lay.ctx[b], n = lay.cu[b + 1] - lay.cu[b];
  const int row_bytes = F8 ? (D == 576 ? 656 : 528) : D * 2;
  uint32_t v[4][9];
  int pos[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = (blockIdx.x & 3) * 32 + i * 8 + warp;
    const int p = pos[i] = blk.y * KT + r;
#pragma unroll
    for (int k = 0; k < 9; ++k) v[i][k] = 0;
    if (p >= c + n) continue;
    const int slot = lay.table[size_t(b) * lay.P + p / lay.page] * lay.page + p % lay.page;
    const uint8_t* src = kv + size_t(slot) * row_bytes;
    if constexpr (F8) {
      const uint4 x = *reinterpret_cast<const uint4*>(src + lane * 16 + (lane >= 16 ? 16 : 0));
      v[i][0] = x.x; v[i][1] = x.y; v[i][2] = x.z; v[i][3] = x.w;
      v[i][4] = src[256 + (lane >> 2)];
      if (D == 576) v[i][8] = reinterpret_cast<const uint32_t*>(src + 528)[lane];
    } else {
      const uint4 x = *reinterpret_cast<const uint4*>(src + lane * 32), y = *reinterpret_cast<const uint4*>(src + lane * 32 + 16);
      v[i][0] = x.x; v[i][1] = x.y; v[i][2] = x.z; v[i][3] = x.w;
      v[i][4] = y.x; v[i][5] = y.y; v[i][6] = y.z; v[i][7] = y.w;
      if (D == 576) v[i][8] = reinterpret_cast<const uint32_t*>(src + 1024)[lane];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t* w = v[i];
    if constexpr (F8) {
      if (pos[i] < c + n) {
        const __half2 sc = __float2half2_rn(ue8m0_to_float(w[4]));
        uint32_t h[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          uint32_t e;
          asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(e) : "h"(uint16_t(w[k >> 1] >> (16 * (k & 1)))));
          const __half2 r = __hmul2(*reinterpret_cast<__half2*>(&e), sc);
          h[k] = *reinterpret_cast<const uint32_t*>(&r);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = h[k];
      }
    }
    if (pos[i] >= c && pos[i] < c + n) {
      const uint32_t expo = F8 ? 0x7C00u : 0x7F80u;
      bool odd = false;
#pragma unroll
      for (int k = 0; k < 9; ++k) odd |= nonfinite16(w[k], expo);
      odd = __any_sync(~0u, odd);
      if (odd)
#pragma unroll
        for (int k = 0; k < 9; ++k) w[k] = 0;
      if (lane == 0) bad[lay.cu[b] + pos[i] - c] = odd;
    }
    const int r = (blockIdx.x & 3) * 32 + i * 8 + warp;
    uint16_t* dst = staged + (size_t(blockIdx.x >> 2) * KT + r) * D;
    *reinterpret_cast<uint4*>(dst + lane * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    *reinterpret_cast<uint4*>(dst + lane * 16 + 8) = make_uint4(w[4], w[5], w[6], w[7]);
    if (D == 576) reinterpret_cast<uint32_t*>(dst + 512)[lane] = w[8];
  }
}

// ---------------------------------------------------------------------------------------------------------------
// The attention kernel.  A stage holds one 128-key tile: chunk a of CTA r = dims [64a, 64a+64) of keys 64r..64r+63,
// what Q·K^T reads as its B operand.  P·V needs, in each CTA, its 256 dims (atoms 4r..4r+3) of all 128 keys: the CTA's
// own keys are there already, the other 64 keys' chunks replace the four chunks that only Q·K^T needed (atoms 4..7 in
// CTA 0, 0..3 in CTA 1), so that both CTAs find keys 0-63 in slots 0-3 and keys 64-127 in slots 4-7, as one
// descriptor has to serve both.  P goes to shared memory (K-major): keys 0-63 over the RoPE chunk (slot 8), keys
// 64-127 into one extra chunk.
//   producer (each CTA)  K(0) K(1) V(0) V(1) | K(2) K(3) V(2) V(3) | ...
//   MMA (CTA 0)          QK(0) QK(1) PV(0) PV(1) | QK(2) QK(3) PV(2) PV(3) | ...
//   softmax (each CTA)   thread = (row, 32 of the 128 keys); the four threads of a row exchange their maxima
// ---------------------------------------------------------------------------------------------------------------
// The tensor maps see a row as 64-dim atoms: (64 dims, rows, atoms), so one TMA load fills several chunks.
struct Maps {
  CUtensorMap q;            // box 64 x 64 rows x all atoms
  CUtensorMap kv4, kv1;     // cache rows: box 64 x Params::box rows x 4 atoms / 1 atom (the RoPE key)
  CUtensorMap st4, st1;     // staged rows: 64 rows
};

template <int NA, bool F16>
__global__ void __launch_bounds__(THREADS, 1) tree_mla_kernel(const __grid_constant__ Maps tm, const Params p) {
#if defined(__CUDA_ARCH__) && __CUDA_ARCH__ >= 1000
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* sQ = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sK = sQ + SLOTS * CH;
  uint8_t* sX = sK + NST * STAGE;                       // P, keys 64-127
  float* xm = reinterpret_cast<float*>(sX + CH);        // [2][256] row maxima (the last tile's buffer, later, sums)
  uint64_t* bars = reinterpret_cast<uint64_t*>(xm + 512);
  uint64_t* q_full = bars;                              // the leader's counts both CTAs' bytes (so do kfull, vfull)
  uint64_t* o_free = bars + 1;                          // leader: both CTAs read the last item's O
  uint64_t* kfull = bars + 2;                           // [NST]
  uint64_t* vfull = kfull + NST;
  uint64_t* sfull = vfull + NST;                        // scores ready (both CTAs)
  uint64_t* p0full = sfull + NST;                       // leader: P of keys 0-63 written, all scores read, O rescaled
  uint64_t* p1full = p0full + NST;                      // leader: P of keys 64-127 written
  uint64_t* pv0 = p1full + NST;                         // P·V of keys 0-63 / 64-127 done (both CTAs)
  uint64_t* pv1 = pv0 + NST;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(pv1 + NST);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  if (sQ + SMEM_USED > smem_raw + SMEM) {                // the same in every CTA
    if (threadIdx.x == 0 && p.status) atomicCAS(p.status, 0, kErrBadArg);
    return;
  }
  const int rank = int(cluster_ctarank());
  const int cluster = blockIdx.x >> 1;
  const uint32_t warp = warp_id(), lane = lane_id();

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(o_free, 2 * SM_WARPS);
    for (int i = 0; i < NST; ++i) {
      mbar_init(&kfull[i], 1); mbar_init(&vfull[i], 1); mbar_init(&sfull[i], 1);
      mbar_init(&p0full[i], 2 * SM_WARPS); mbar_init(&p1full[i], SM_WARPS); mbar_init(&pv0[i], 1); mbar_init(&pv1[i], 1);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 2) { tmem_alloc_pair(tmem_slot, 512); tmem_relinquish_pair(); }
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_entry();
  const int i0 = p.work.first[cluster], i1 = p.work.first[cluster + 1];
  auto fail = [&](int code) { if (p.status) atomicCAS(p.status, 0, code); *abort_flag = 1; };
  auto wait = [&](uint64_t* bar, uint32_t phase, int code) -> bool {
    if (mbar_wait(bar, phase)) return true;
    fail(code);
    return false;
  };

  if (warp == 0) {
    // ---------------- producer ----------------
    if (lane == 0) {
      tma_prefetch_desc(&tm.q); tma_prefetch_desc(&tm.kv4); tma_prefetch_desc(&tm.kv1);
      tma_prefetch_desc(&tm.st4); tma_prefetch_desc(&tm.st1);
      const uint32_t lead_q = mapa_shared(smem_u32(q_full), 0);
      int g = 0;                                        // tiles so far: stage g % 2, phase (g / 2) & 1
      bool ok = true;
      for (int i = i0; ok && i < i1; ++i) {
        const TreeItem it = p.work.items[i];
        const int ctx = p.lay.ctx[it.b];
        const int staged_from = p.stage_all ? 0 : ctx / KT;
        const int* table = p.lay.table + size_t(it.b) * p.lay.P;
        // n atoms from atom a of 64 keys (half `half` of a tile) -> chunks.  The first rows of a tile's boxes are looked
        // up ahead of the waits: a page-table read per load would cost more than the load's issue.
        auto row_of = [&](int tile, int half, int r) -> int {
          if (tile >= staged_from) return (p.work.stage_at[it.b] + tile - staged_from) * KT + half * 64 + r;
          const int pos = tile * KT + half * 64 + r;
          return table[pos / p.lay.page] * p.lay.page + pos % p.lay.page;
        };
        auto load = [&](uint8_t* dst, uint32_t bar, int tile, int half, int row0, int a, bool four) {
          if (tile >= staged_from) {
            tma_load_3d_pair(dst, four ? &tm.st4 : &tm.st1, bar, 0, row0, a);
          } else if (p.box == 64) {
            tma_load_3d_pair(dst, four ? &tm.kv4 : &tm.kv1, bar, 0, row0, a);
          } else {              // a box shorter than a chunk: one atom at a time
            for (int r = 0; r < 64; r += p.box) {
              const int row = r ? row_of(tile, half, r) : row0;
              for (int k = 0; k < (four ? 4 : 1); ++k)
                tma_load_3d_pair(dst + k * CH + r * 128, &tm.kv1, bar, 0, row, a + k);
            }
          }
        };
        // L2 prefetch of the CTA's half of a tile two tiles before its load: the ring holds two tiles, too few to cover
        // the latency of HBM
        auto prefetch = [&](int tile) {
          if (tile >= staged_from || p.box != 64) return;
          const int row = row_of(tile, rank, 0);
          tma_prefetch_l2_3d(&tm.kv4, 0, row, 0);
          tma_prefetch_l2_3d(&tm.kv4, 0, row, 4);
          if (NA == 9) tma_prefetch_l2_3d(&tm.kv1, 0, row, 8);
        };
        // Q: the previous item's last Q·K^T is done (its V loads waited for it)
        if (rank == 0) mbar_arrive_expect_tx(q_full, 2 * NA * CH);
        const int q_row = p.lay.cu[it.b] * p.H + it.row * 128 + rank * 64;
        tma_load_3d_pair(sQ, &tm.q, lead_q, 0, q_row, 0);
        for (int j = 0; ok && j < it.n_tiles; j += 2) {
          const int m = min(2, it.n_tiles - j);
          for (int u = 0; ok && u < m; ++u) {
            const int s = (g + u) & 1, ph = ((g + u) >> 1) & 1;
            uint8_t* st = sK + s * STAGE;
            const uint32_t bar = mapa_shared(smem_u32(&kfull[s]), 0);
            const int tile = it.tile + j + u, row0 = row_of(tile, rank, 0);
            if (rank == 0) mbar_arrive_expect_tx(&kfull[s], 2 * NA * CH);
            if (!(ok = wait(&pv0[s], ph ^ 1, kErrTimeoutEmpty))) break;
            load(st, bar, tile, rank, row0, 0, true);
            if (NA == 9) load(st + 8 * CH, bar, tile, rank, row0, 8, false);
            if (!(ok = wait(&pv1[s], ph ^ 1, kErrTimeoutEmpty))) break;
            load(st + 4 * CH, bar, tile, rank, row0, 4, true);
            if (j + u + 2 < it.n_tiles) prefetch(tile + 2);
          }
          for (int u = 0; ok && u < m; ++u) {
            const int s = (g + u) & 1, ph = ((g + u) >> 1) & 1;
            uint8_t* st = sK + s * STAGE;
            const uint32_t bar = mapa_shared(smem_u32(&vfull[s]), 0);
            const int tile = it.tile + j + u, row0 = row_of(tile, rank ^ 1, 0);
            if (rank == 0) mbar_arrive_expect_tx(&vfull[s], 2 * 4 * CH);
            if (!(ok = wait(&sfull[s], ph, kErrTimeoutFull))) break;
            load(st + (rank ? 0 : 4) * CH, bar, tile, rank ^ 1, row0, 4 * rank, true);
          }
          g += m;
        }
        if (*abort_flag) ok = false;
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA (the leader issues for both CTAs) ----------------
    if (rank == 0 && elect_one()) {
      const uint32_t id_qk = F16 ? idesc_f16(128, KT) : idesc_bf16(128, KT);
      const uint32_t id_pv = (F16 ? idesc_f16(128, 256) : idesc_bf16(128, 256)) | (1u << 16);   // V is MN-major
      int g = 0;
      bool ok = true;
      for (int i = i0; ok && i < i1; ++i) {
        const int nt = p.work.items[i].n_tiles;
        ok = wait(q_full, (i - i0) & 1, kErrTimeoutFull);
        for (int j = 0; ok && j < nt; j += 2) {
          const int m = min(2, nt - j);
          for (int u = 0; ok && u < m; ++u) {
            const int s = (g + u) & 1, ph = ((g + u) >> 1) & 1;
            const uint8_t* st = sK + s * STAGE;
            if (!(ok = wait(&kfull[s], ph, kErrTimeoutFull))) break;
            tc_fence_after();
            for (int a = 0; a < NA; ++a)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                mma_f16_ss_pair(tmem + TM_S + s * 64, smem_desc_sw128(sQ + a * CH + k * 32),
                                smem_desc_sw128(st + a * CH + k * 32), id_qk, (a | k) > 0);
            mma_commit_pair(&sfull[s], 3);
          }
          for (int u = 0; ok && u < m; ++u) {
            const int s = (g + u) & 1, ph = ((g + u) >> 1) & 1;
            const uint8_t* st = sK + s * STAGE;
            if (j + u == 0 && i > i0) ok = wait(o_free, (i - i0 - 1) & 1, kErrTimeoutTmem);
            ok = ok && wait(&vfull[s], ph, kErrTimeoutFull) && wait(&p0full[s], ph, kErrTimeoutTmem);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint64_t a = smem_desc_sw128(st + 8 * CH + k * 32);
              const uint32_t acc = (j + u > 0 || k > 0) ? 1u : 0u;
              mma_f16_ss_pair_keep_a(tmem + TM_O, a, desc_mn(st + k * 2048), id_pv, acc);
              mma_f16_ss_pair_last_a(tmem + TM_O + 128, a, desc_mn(st + 2 * CH + k * 2048), id_pv, acc);
            }
            mma_commit_pair(&pv0[s], 3);
            if (!(ok = wait(&p1full[s], ph, kErrTimeoutTmem))) break;
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint64_t a = smem_desc_sw128(sX + k * 32);
              mma_f16_ss_pair_keep_a(tmem + TM_O, a, desc_mn(st + 4 * CH + k * 2048), id_pv, 1u);
              mma_f16_ss_pair_last_a(tmem + TM_O + 128, a, desc_mn(st + 6 * CH + k * 2048), id_pv, 1u);
            }
            mma_commit_pair(&pv1[s], 3);
          }
          g += m;
          if (*abort_flag) ok = false;
        }
      }
    }
  } else if (warp >= 4) {
    // ---------------- softmax, rescale, epilogue: lanes 0-63 / 64-127 hold the first / second 64 keys of the rows;
    // two warps share 32 lanes and take 32 score columns (and 128 of the 256 columns of O) each -------
    const int q = warp & 3, half = q >> 1, row = (q & 1) * 32 + int(lane), part = (int(warp) - 4) >> 2;
    const int me = part * 128 + q * 32 + int(lane);
    const uint32_t t_lane = tmem + (uint32_t(q * 32) << 16);
    int g = 0;
    bool ok = true;                       // after a failed wait the loop runs on without waiting: the block-level
    for (int i = i0; i < i1; ++i) {       // barriers below need all the warps
      const TreeItem it = p.work.items[i];
      const int ctx = p.lay.ctx[it.b], c0 = p.lay.cu[it.b], n = p.lay.cu[it.b + 1] - c0;
      const int r = it.row * 128 + rank * 64 + row;
      const bool live = r < n * p.H;
      const int node = live ? r / p.H : 0, head = r - node * p.H;
      const uint64_t mask = live ? uint64_t(p.mask[c0 + node]) : 0;
      float m_used = -INFINITY, l = 0.f;
      for (int j = 0; j < it.n_tiles; ++j, ++g) {
        const int s = g & 1, ph = (g >> 1) & 1;
        ok = ok && wait(&sfull[s], ph, kErrTimeoutTmem);
        tc_fence_after();
        uint32_t x[32];
        tmem_ld_32x32b_x32(t_lane + TM_S + s * 64 + part * 32, x);
        tmem_ld_wait();
        const int first = (it.tile + j) * KT + half * 64 + part * 32;   // position of this thread's first key
        if (first + 32 > ctx) {
          const int off = ctx - first;                                  // keys before the tree
          const uint32_t pre = off <= 0 ? 0 : (1u << off) - 1;
          const uint32_t see = pre | uint32_t(off >= 0 ? mask << off : (off > -64 ? mask >> -off : 0));
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if (!((see >> k) & 1)) x[k] = 0xff800000u;
        }
        float m0 = -INFINITY, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          m0 = fmaxf(m0, __uint_as_float(x[k])); m1 = fmaxf(m1, __uint_as_float(x[k + 1]));
          m2 = fmaxf(m2, __uint_as_float(x[k + 2])); m3 = fmaxf(m3, __uint_as_float(x[k + 3]));
        }
        float* xb = xm + (g & 1) * 256;
        xb[me] = fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
        softmax_sync();
        const float mt = fmaxf(fmaxf(xb[me], xb[me ^ 64]), fmaxf(xb[me ^ 128], xb[me ^ 192])) * p.scale_log2;
        const bool grow = j > 0 && mt > m_used + kRescale;
        const float m_new = grow || j == 0 ? fmaxf(m_used, mt) : m_used;
        const float m_ref = m_new == -INFINITY ? 0.f : m_new;
        if (__any_sync(~0u, grow)) {
          const float keep = grow && m_used != -INFINITY ? ex2(m_used - m_ref) : 1.f;
          ok = ok && wait(&pv1[s ^ 1], ((g - 1) >> 1) & 1, kErrTimeoutTmem);
          tc_fence_after();
#pragma unroll 1
          for (int c = part * 128; c < part * 128 + 128; c += 32) {
            uint32_t o[32];
            tmem_ld_32x32b_x32(t_lane + TM_O + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * keep);
            tmem_st_32x32b_x32(t_lane + TM_O + c, o);
          }
          tmem_st_wait();
          l *= keep;
        }
        m_used = m_new;
        float l0 = 0.f, l1 = 0.f;
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          const float a = ex2(fmaf(__uint_as_float(x[k]), p.scale_log2, -m_ref));
          const float b = ex2(fmaf(__uint_as_float(x[k + 1]), p.scale_log2, -m_ref));
          l0 += a;
          l1 += b;
          x[k / 2] = pack2(a, b, F16);
        }
        l += l0 + l1;
        tc_fence_before();
        if (half) {
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&p0full[s]), 0));   // scores read, O rescaled
          // the extra chunk: the previous tile's P·V must have read it
          ok = ok && wait(&pv1[s ^ 1], ((g - 1) >> 1) & 1, kErrTimeoutTmem);
        }
        uint8_t* dst = (half ? sX : sK + s * STAGE + 8 * CH) + row * 128;
#pragma unroll
        for (int c = 0; c < 4; ++c)
          *reinterpret_cast<uint4*>(dst + (((part * 4 + c) ^ (row & 7)) << 4)) =
              make_uint4(x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(half ? &p1full[s] : &p0full[s]), 0));
      }
      // ---- item's end
      const int sl = (g - 1) & 1;
      ok = ok && wait(&pv1[sl], ((g - 1) >> 1) & 1, kErrTimeoutTmem);
      tc_fence_after();
      if ((it.tile + it.n_tiles) * KT > ctx) {            // nodes that see a marked row become NaN
        const int b0 = int(lane) < n ? p.bad[c0 + lane] : 0, b1 = int(lane) + 32 < n ? p.bad[c0 + 32 + lane] : 0;
        const uint64_t bad = uint64_t(__ballot_sync(~0u, b0)) | uint64_t(__ballot_sync(~0u, b1)) << 32;
        if (mask & bad) l = __int_as_float(0x7fffffff);
      }
      // sums: the maxima buffer of the tile before last is free, and the next item's first tile takes it only after
      // every warp passed the second barrier
      float* xs = xm + (g & 1) * 256;
      xs[me] = l;
      softmax_sync();
      l = (xs[me] + xs[me ^ 64]) + (xs[me ^ 128] + xs[me ^ 192]);
      softmax_sync();
      float inv = 1.f;
      if (it.part < 0) {
        if (p.sink && live) l += exp2f(p.sink[head] * 1.4426950408889634f - (m_used == -INFINITY ? 0.f : m_used));
        inv = l == 0.f ? 0.f : 1.f / l;
      } else if (half == 0 && part == 0) {
        float* ml = p.part_ml + (size_t(it.part) * 128 + rank * 64 + row) * 2;
        ml[0] = m_used;
        ml[1] = l;
      }
      __nv_bfloat16* o = p.out + (size_t(c0) * p.H + r) * 512 + half * 256 + part * 128;
      float* po = p.part_o + (size_t(max(it.part, 0)) * 128 + rank * 64 + row) * 512 + half * 256 + part * 128;
#pragma unroll 1
      for (int c = 0; c < 128; c += 32) {
        uint32_t v[32];
        tmem_ld_32x32b_x32(t_lane + TM_O + part * 128 + c, v);
        tmem_ld_wait();
        if (it.part >= 0) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            reinterpret_cast<uint4*>(po + c)[k] = make_uint4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
        } else if (live) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            reinterpret_cast<uint4*>(o + c)[k] =
                make_uint4(pack_bf16x2(__uint_as_float(v[8 * k]) * inv, __uint_as_float(v[8 * k + 1]) * inv),
                           pack_bf16x2(__uint_as_float(v[8 * k + 2]) * inv, __uint_as_float(v[8 * k + 3]) * inv),
                           pack_bf16x2(__uint_as_float(v[8 * k + 4]) * inv, __uint_as_float(v[8 * k + 5]) * inv),
                           pack_bf16x2(__uint_as_float(v[8 * k + 6]) * inv, __uint_as_float(v[8 * k + 7]) * inv));
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(o_free), 0));
    }
  }
  __syncthreads();
  if (*abort_flag)                        // a wait ran out: let copies in flight land before the memory is given up
    for (int i = 0; i < 100; ++i) __nanosleep(1000);
  cluster_sync();
  if (warp == 2) { tc_fence_after(); tmem_dealloc_pair(tmem, 512); }
#endif
}

// out = sum_s 2^(m_s - M) O_s / (sum_s 2^(m_s - M) l_s + sink): one CTA per row of a split row tile, four of the 512
// dims per thread, eight partial rows in flight.
__global__ void __launch_bounds__(128) tree_merge_kernel(TreeLayout lay, const TreeMerge* __restrict__ merges, int H,
                                                         const float* __restrict__ part_o,
                                                         const float* __restrict__ part_ml,
                                                         const float* __restrict__ sink,
                                                         __nv_bfloat16* __restrict__ out) {
  pdl_entry();
  const TreeMerge mg = merges[blockIdx.x];
  const int row = blockIdx.y;
  const int r = mg.row * 128 + row, n = lay.cu[mg.b + 1] - lay.cu[mg.b];
  if (r >= n * H) return;
  const float2* ml = reinterpret_cast<const float2*>(part_ml) + size_t(mg.part) * 128 + row;
  const float sk = sink ? sink[r % H] * 1.4426950408889634f : -INFINITY;
  float M = sk;
#pragma unroll 8
  for (int s = 0; s < mg.n; ++s) M = fmaxf(M, ml[s * 128].x);
  if (M == -INFINITY) M = 0.f;
  float L = exp2f(sk - M);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  const float4* po = reinterpret_cast<const float4*>(part_o) + (size_t(mg.part) * 128 + row) * 128 + threadIdx.x;
#pragma unroll 8
  for (int s = 0; s < mg.n; ++s) {
    const float2 v = ml[s * 128];
    const float4 o = po[size_t(s) * 128 * 128];
    const float w = exp2f(v.x - M);
    L += w * v.y;
    acc.x += w * o.x; acc.y += w * o.y; acc.z += w * o.z; acc.w += w * o.w;
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  reinterpret_cast<uint2*>(out + (size_t(lay.cu[mg.b]) * H + r) * 512)[threadIdx.x] =
      make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
}

static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    const bool ok = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000, cudaEnableDefault, &q) ==
                        cudaSuccess && q == cudaDriverEntryPointSuccess;
    return ok ? reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr) : nullptr;
  }();
  return fn;
}

// [rows, D] 16-bit row-major matrix as (64, rows, D / 64), read in boxes of 64 x box_rows x atoms
static bool row_map(CUtensorMap* m, bool f16, const void* base, int64_t rows, int D, int box_rows, int atoms) {
  const cuuint64_t dims[3] = {64, cuuint64_t(rows), cuuint64_t(D) / 64};
  const cuuint64_t str[2] = {cuuint64_t(D) * 2, 128};
  const cuuint32_t box[3] = {64, cuuint32_t(box_rows), cuuint32_t(atoms)}, es[3] = {1, 1, 1};
  return encode_fn()(m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                     const_cast<void*>(base), dims, str, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

using Kernel = void (*)(const Maps, const Params);

static cudaLaunchConfig_t pair_config(int clusters, cudaLaunchAttribute* attr, cudaStream_t s) {
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * clusters);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cfg;
}

}  // namespace tree

int tree_mla_clusters() {
  tree::Kernel f = tree::tree_mla_kernel<9, false>;
  if (smem_optin(f, tree::SMEM) != cudaSuccess) return 0;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = tree::pair_config(1, attr, nullptr);
  cfg.numAttrs = 1;
  int n = 0;
  return cudaOccupancyMaxActiveClusters(&n, f, &cfg) == cudaSuccess ? n : 0;
}

cudaError_t tree_mla(const void* q, int T, int H, int D, bool f8, bool all, const void* kv, int64_t S,
                     const TreeLayout& lay, const TreeWork& work, const int64_t* mask, float scale, const float* sink,
                     void* staged, int* bad, float* part_o, float* part_ml, int* status, void* out, cudaStream_t s) {
  using namespace tree;
  if (!encode_fn()) return cudaErrorNotSupported;
  if (D != 576 && D != 512) return cudaErrorInvalidValue;
  int box = 64;
  while (lay.page % box) box /= 2;
  if (box < 8 && !all) return cudaErrorInvalidValue;
  Maps m;
  const int64_t st_rows = int64_t(work.n_stage) * KT;
  if (!row_map(&m.q, f8, q, int64_t(T) * H, D, 64, D / 64) || !row_map(&m.st4, f8, staged, st_rows, D, 64, 4) ||
      !row_map(&m.st1, f8, staged, st_rows, D, 64, 1))
    return cudaErrorInvalidValue;
  m.kv4 = m.st4;
  m.kv1 = m.st1;
  if (!all && !(row_map(&m.kv4, false, kv, S, D, box, 4) && row_map(&m.kv1, false, kv, S, D, box, 1)))
    return cudaErrorInvalidValue;
  const auto* kvb = reinterpret_cast<const uint8_t*>(kv);
  auto* st = reinterpret_cast<uint16_t*>(staged);
  cudaError_t e = launch_k(f8 ? tree_stage_kernel<true> : tree_stage_kernel<false>, dim3(work.n_stage * 4), 256, 0, s,
                           kvb, lay, work.stage, D, st, bad);
  if (e != cudaSuccess) return e;
  Params p;
  p.lay = lay; p.work = work; p.mask = mask; p.bad = bad;
  p.H = H; p.stage_all = all; p.box = box;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.sink = sink; p.part_o = part_o; p.part_ml = part_ml; p.status = status;
  p.out = reinterpret_cast<__nv_bfloat16*>(out);
  Kernel f = D == 576 ? (f8 ? tree_mla_kernel<9, true> : tree_mla_kernel<9, false>)
                      : (f8 ? tree_mla_kernel<8, true> : tree_mla_kernel<8, false>);
  if ((e = smem_optin(f, SMEM)) != cudaSuccess) return e;
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = pair_config(work.clusters, attr, s);
  if ((e = cudaLaunchKernelEx(&cfg, f, m, p)) != cudaSuccess || !work.n_merges) return e;
  return launch_k(tree_merge_kernel, dim3(work.n_merges, 128), 128, 0, s, lay, work.merges, H, part_o, part_ml, sink,
                  p.out);
}

}  // namespace cb
