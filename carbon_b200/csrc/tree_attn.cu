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
// Key tiles come into shared memory by TMA where they lie there as the tensor core reads them: whole tiles of bf16 rows
// in pages of a multiple of 64, or rows that tree_stage_kernel has expanded to dense fp16 / bf16 first (fp8 rows and other
// pages, in calls large enough to read them twice).  Else such rows, and each request's last tiles always (which end, or
// belong to the tree), are fed by warps: global memory -> registers -> fp16 / bf16 in the swizzled layout.
// tree_merge_kernel joins row tiles whose keys were split over CTA pairs.
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
constexpr int FEED_WARPS = 8;              // eight rows (one swizzle group) of a CTA's 64 keys each
constexpr int THREADS = 64 + FEED_WARPS * 32 + SM_WARPS * 32;
constexpr int SMEM_USED = SLOTS * CH + NST * STAGE + CH + 2048 + 256;
constexpr int SMEM = SMEM_USED + 768;      // 227 KB; the base is 256-byte aligned at least (checked by the kernel)
constexpr float kRescale = 8.f;            // O is rescaled when the running maximum grows by more than 2^8

enum { FEED, PAGED, STAGED };
struct Params {
  TreeLayout lay;
  TreeWork work;
  const int64_t* mask;
  const uint8_t* kv;
  int H, how;                              // how whole tiles come: FEED, PAGED or STAGED
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
CB_DEVICE void store32(void* p, const uint32_t* v) {      // one 32-byte sector (p 32-byte aligned)
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
// Four lanes (rows) x four units of eight words: afterwards unit u of lane j is unit j of the lane u of its four.  Rows
// that each lane holds for itself become 128-byte runs of one row over four lanes.
CB_DEVICE void quad_transpose(uint32_t (&v)[32], int lane) {
#pragma unroll
  for (int step = 1; step <= 2; step *= 2) {
    const bool up = lane & step;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (u & step) continue;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t got = __shfl_xor_sync(~0u, up ? v[8 * u + k] : v[8 * (u + step) + k], step);
        if (up) v[8 * u + k] = got;
        else v[8 * (u + step) + k] = got;
      }
    }
  }
}
CB_DEVICE void softmax_sync() { asm volatile("bar.sync 1, %0;" ::"n"(SM_WARPS * 32) : "memory"); }

// ---------------------------------------------------------------------------------------------------------------
// Feeding: a warp brings eight rows into swizzled chunks.  Row r of the CTA's 64, 16-byte piece c of atom a goes to
// chunk a, byte r * 128 + ((c ^ (r & 7)) << 4).
// ---------------------------------------------------------------------------------------------------------------
template <bool F8>
CB_DEVICE bool odd16(const uint4& v) {       // a NaN or an infinity among eight fp16 (F8) / bf16 values
  constexpr uint32_t e = F8 ? 0x7C00u : 0x7F80u;
  auto bad = [](uint32_t w) { return (w & e) == e || ((w >> 16) & e) == e; };
  return bad(v.x) | bad(v.y) | bad(v.z) | bad(v.w);
}
// 16 e4m3 values and their atom's UE8M0 scale -> 16 fp16 (exact while the products fit fp16)
CB_DEVICE void expand16(const uint4& v, uint32_t scale, uint4& a, uint4& b) {
  const __half2 sc = __float2half2_rn(ue8m0_to_float(scale));
  uint32_t h[8];
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    uint32_t e;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(e) : "h"(uint16_t(w[k >> 1] >> (16 * (k & 1)))));
    const __half2 r = __hmul2(*reinterpret_cast<__half2*>(&e), sc);
    h[k] = *reinterpret_cast<const uint32_t*>(&r);
  }
  a = make_uint4(h[0], h[1], h[2], h[3]);
  b = make_uint4(h[4], h[5], h[6], h[7]);
}
CB_DEVICE void put(uint8_t* chunk, int row, int c, const uint4& v) {
  *reinterpret_cast<uint4*>(chunk + row * 128 + ((c ^ (row & 7)) << 4)) = v;
}

// Whole key tiles -> dense fp16 / bf16 rows.  A CTA brings 32 rows, a warp four.  Bound by HBM: 103,000 fp8 rows in 33 us
// (5.6 TB/s read and written).
template <bool F8>
__global__ void __launch_bounds__(256) tree_stage_kernel(const uint8_t* __restrict__ kv, TreeLayout lay,
                                                         const int2* __restrict__ blocks, int D,
                                                         uint16_t* __restrict__ staged) {
  pdl_entry();
  const int lane = threadIdx.x & 31, r0 = (blockIdx.x & 3) * 32 + (threadIdx.x >> 5) * 4;
  const int2 blk = blocks[blockIdx.x >> 2];
  const int pos = blk.y * KT + r0 + (lane & 3);
  const int mine = lay.table[size_t(blk.x) * lay.P + pos / lay.page] * lay.page + pos % lay.page;
  const int row_bytes = F8 ? (D == 576 ? 656 : 528) : D * 2;
  uint4 v[4], w[4];
  uint32_t pe[4], sc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint8_t* src = kv + int64_t(__shfl_sync(~0u, mine, i)) * row_bytes;
    if constexpr (F8) {
      v[i] = reinterpret_cast<const uint4*>(src)[lane + (lane >= 16 ? 1 : 0)];
      sc[i] = src[256 + (lane >> 2)];
    } else {
      v[i] = reinterpret_cast<const uint4*>(src)[2 * lane];
      w[i] = reinterpret_cast<const uint4*>(src)[2 * lane + 1];
    }
    pe[i] = D == 576 ? reinterpret_cast<const uint32_t*>(src + (F8 ? 528 : 1024))[lane] : 0;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (F8) {
      uint4 a;
      expand16(v[i], sc[i], a, w[i]);
      v[i] = a;
    }
    uint16_t* dst = staged + (size_t(blockIdx.x >> 2) * KT + r0 + i) * D;
    reinterpret_cast<uint4*>(dst)[2 * lane] = v[i];
    reinterpret_cast<uint4*>(dst)[2 * lane + 1] = w[i];
    if (D == 576) reinterpret_cast<uint32_t*>(dst + 512)[lane] = pe[i];
  }
}

// ---------------------------------------------------------------------------------------------------------------
// The attention kernel.  A stage holds one 128-key tile: chunk a of CTA r = dims [64a, 64a+64) of keys 64r..64r+63,
// what Q·K^T reads as its B operand.  P·V needs, in each CTA, its 256 dims (atoms 4r..4r+3) of all 128 keys: the CTA's
// own keys are there already, the other 64 keys' chunks replace the four chunks that only Q·K^T needed (atoms 4..7 in
// CTA 0, 0..3 in CTA 1), so that both CTAs find keys 0-63 in slots 0-3 and keys 64-127 in slots 4-7, as one
// descriptor has to serve both.  P goes to shared memory (K-major): keys 0-63 over the RoPE chunk (slot 8), keys
// 64-127 into one extra chunk.
//   producer, feed (each CTA)  K(0) K(1) V(0) V(1) | K(2) K(3) V(2) V(3) | ...
//   MMA (CTA 0)          QK(0) QK(1) PV(0) PV(1) | QK(2) QK(3) PV(2) PV(3) | ...
//   softmax (each CTA)   thread = (row, 32 of the 128 keys); the four threads of a row exchange their maxima
// Probabilities enter P·V as bf16 (fp16 for fp8 rows), the rows' own rounding: their errors average out over the keys
// (relative error of the output 2.1e-3 against 1.7e-3 of rounding it alone).  Scores, maxima, sums and O are fp32.
//
// What bounds it: a 128-key tile is 128 x 128 x 1088 MACs, 2176 cycles of a pair's tensor cores; it takes 2.06 us with
// the keys in L2 (1.28 PFLOP/s, 64 tiles on 74 pairs), 2.7 us with 32 tiles per pair from HBM.  The ring holds two
// tiles (Q 72 KB, 2 x 72 KB of keys, P), so the matrix instructions of one tile cover the softmax of the other only
// partly (tensor pipe 66 % active): its 1,600 cycles of latency are 60 loading and 180 for the maximum, 320 exchanging
// it, 660 exponentials (16 a cycle), 380 storing P and its proxy fence, and the barriers to and from the issuing thread
// add 1,200.  Large calls run into the power cap first (1.57 GHz at 1.1 PFLOP/s).
// ---------------------------------------------------------------------------------------------------------------
// A fed row with a NaN or an infinity in a tile that holds tree rows: Q·K^T sees it (its scores are NaN, and so is every
// node that sees it), but the values P·V multiplies by a weight of zero for the other branches' nodes are made zero.
//
// Arrives at the leader's barriers from the other CTA have the default scope, the CTA's.  What they announce stays in the
// arriving warp's own SM: its shared memory (after the proxy fence) and TMEM, which that SM's tensor core reads when the
// leader issues for the pair.  Nothing has to become visible to another SM first, and a release to the cluster's scope
// before each arrive took 3.0 us a tile instead of 2.07.
//
// The tensor maps see a row as 64-dim atoms: (64 dims, rows, atoms), so one TMA load fills several chunks.
struct Maps {
  CUtensorMap q;            // box 64 x 64 rows x all atoms
  CUtensorMap kv4, kv1;     // cache rows or staged rows: box 64 x 64 rows x 4 atoms / 1 atom (the RoPE key)
};

template <int NA, bool F16>
__global__ void __launch_bounds__(THREADS, 1) tree_mla_kernel(const __grid_constant__ Maps tm, const Params p) {
#if defined(__CUDA_ARCH__) && __CUDA_ARCH__ >= 1000
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* sQ = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sK = sQ + SLOTS * CH;
  uint8_t* sX = sK + NST * STAGE;                       // P, keys 64-127
  float* xm = reinterpret_cast<float*>(sX + CH);        // [2][256] row maxima, at an item's end sums
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
      // the producer of CTA 0 and the feed warps of both CTAs arrive for every tile
      mbar_init(&kfull[i], 1 + 2 * FEED_WARPS); mbar_init(&vfull[i], 1 + 2 * FEED_WARPS); mbar_init(&sfull[i], 1);
      mbar_init(&p0full[i], 2 * SM_WARPS); mbar_init(&p1full[i], SM_WARPS); mbar_init(&pv0[i], 1); mbar_init(&pv1[i], 1);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 2) { tmem_alloc_pair(tmem_slot, 512); tmem_relinquish_pair(); }
  const int i0 = p.work.first[cluster], i1 = p.work.first[cluster + 1];   // made by the host: no kernel writes them
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // Items and page table are made by the host: the roles look up their first rows before they wait for the kernel that
  // wrote the queries and the cache.
  pdl_launch_dependents();
  auto fail = [&](int code) { if (p.status) atomicCAS(p.status, 0, code); *abort_flag = 1; };
  auto wait = [&](uint64_t* bar, uint32_t phase, int code) -> bool {
    if (mbar_wait(bar, phase)) return true;
    fail(code);
    return false;
  };

  // whether a key tile comes by TMA
  auto by_tma = [&](const TreeItem& it, int tile) { return p.how != FEED && (tile + 1) * KT <= it.ctx; };

  if (warp == 0) {
    // ---------------- producer: Q and the key tiles that TMA can take ----------------
    if (lane == 0) {
      tma_prefetch_desc(&tm.q); tma_prefetch_desc(&tm.kv4); tma_prefetch_desc(&tm.kv1);
      const uint32_t lead_q = mapa_shared(smem_u32(q_full), 0);
      int g = 0;                                        // tiles so far: stage g % 2, phase (g / 2) & 1
      bool ok = true;
      TreeItem nx = p.work.items[i0];                   // items are read one ahead
      for (int i = i0; ok && i < i1; ++i) {
        const TreeItem it = nx;
        if (i + 1 < i1) nx = p.work.items[i + 1];
        auto row_in = [&](const TreeItem& t, int tile, int half) -> int {   // row of a half tile's first key
          const int pos = tile * KT + half * 64;
          if (p.how == STAGED) return p.work.stage_at[t.b] * KT + pos;
          return p.lay.table[size_t(t.b) * p.lay.P + pos / p.lay.page] * p.lay.page + pos % p.lay.page;
        };
        auto row_of = [&](int tile, int half) { return row_in(it, tile, half); };
        if (i == i0) pdl_wait();
        // Q: the previous item's last Q·K^T is done (its V loads waited for it)
        if (rank == 0) mbar_arrive_expect_tx(q_full, 2 * NA * CH);
        tma_load_3d_pair(sQ, &tm.q, lead_q, 0, it.c0 * p.H + it.row * 128 + rank * 64, 0);
        for (int j = 0; ok && j < it.n_tiles; j += 2) {
          const int m = min(2, it.n_tiles - j);
          for (int u = 0; ok && u < m; ++u) {
            const int s = (g + u) & 1, ph = ((g + u) >> 1) & 1, tile = it.tile + j + u;
            const bool tma = by_tma(it, tile);
            uint8_t* st = sK + s * STAGE;
            const uint32_t bar = mapa_shared(smem_u32(&kfull[s]), 0);
            const int row = tma ? row_of(tile, rank) : 0;       // looked up ahead of the waits
            if (!(ok = wait(&pv0[s], ph ^ 1, kErrTimeoutEmpty))) break;
            if (rank == 0) {
              if (tma) mbar_arrive_expect_tx(&kfull[s], 2 * NA * CH);
              else mbar_arrive(&kfull[s]);
            }
            if (tma) {
              tma_load_3d_pair(st, &tm.kv4, bar, 0, row, 0);
              if (NA == 9) tma_load_3d_pair(st + 8 * CH, &tm.kv1, bar, 0, row, 8);
            }
            if (!(ok = wait(&pv1[s], ph ^ 1, kErrTimeoutEmpty))) break;
            if (tma) tma_load_3d_pair(st + 4 * CH, &tm.kv4, bar, 0, row, 4);
            // L2 prefetch of the CTA's half two tiles on: the ring holds two tiles, too few to cover the latency of HBM
            int r2 = -1;
            if (j + 2 < it.n_tiles) {
              if (j + u + 2 < it.n_tiles && by_tma(it, tile + 2)) r2 = row_of(tile + 2, rank);
            } else if (i + 1 < i1 && u < nx.n_tiles && by_tma(nx, nx.tile + u)) {
              r2 = row_in(nx, nx.tile + u, rank);
            }
            if (r2 >= 0) {
              tma_prefetch_l2_3d(&tm.kv4, 0, r2, 0);
              tma_prefetch_l2_3d(&tm.kv4, 0, r2, 4);
              if (NA == 9) tma_prefetch_l2_3d(&tm.kv1, 0, r2, 8);
            }
          }
          for (int u = 0; ok && u < m; ++u) {
            const int s = (g + u) & 1, ph = ((g + u) >> 1) & 1, tile = it.tile + j + u;
            const bool tma = by_tma(it, tile);
            const int row = tma ? row_of(tile, rank ^ 1) : 0;
            if (!(ok = wait(&sfull[s], ph, kErrTimeoutFull))) break;
            if (rank == 0) {
              if (tma) mbar_arrive_expect_tx(&vfull[s], 2 * 4 * CH);
              else mbar_arrive(&vfull[s]);
            }
            if (tma)
              tma_load_3d_pair(sK + s * STAGE + (rank ? 0 : 4) * CH, &tm.kv4, mapa_shared(smem_u32(&vfull[s]), 0), 0,
                               row, 4 * rank);
          }
          g += m;
        }
        if (*abort_flag) ok = false;
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA (the leader issues for both CTAs) ----------------
    pdl_wait();
    if (rank == 0 && elect_one()) {
      const uint32_t id_qk = F16 ? idesc_f16(128, KT) : idesc_bf16(128, KT);
      const uint32_t id_pv = (F16 ? idesc_f16(128, 256) : idesc_bf16(128, 256)) | (1u << 16);   // V is MN-major
      int g = 0, next_nt = p.work.items[i0].n_tiles;
      bool ok = true;
      for (int i = i0; ok && i < i1; ++i) {
        const int nt = next_nt;
        if (i + 1 < i1) next_nt = p.work.items[i + 1].n_tiles;
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
  } else if (warp < 2 + FEED_WARPS) {
    // ---------------- feed: rows r0 .. r0 + 7 of the CTA's 64 keys (K) and of the peer's (V) ----------------
    // A tile's loads are issued before the wait for its slots; the slots' cache rows were looked up a pair of tiles
    // earlier (a dependent page-table read per tile would cost as much as the conversion).  A fed fp8 tile takes 4.0 us:
    // one warp's rows go through waiting, converting and storing in turn (2,100 cycles for K, 1,200 for V, twice a
    // pair).  Eight values per load instead of sixteen needs fewer instructions but more loads and was 5 % slower.
    constexpr bool F8 = F16;
    constexpr int RB = F8 ? (NA == 9 ? 656 : 528) : NA * 128;
    const int r0 = (int(warp) - 2) * 8;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    int g = 0;
    bool ok = true;
    // cache rows of a pair of tiles, one lookup by the whole warp: lanes 0-7 and 8-15 hold those of rows r0 .. r0 + 7 of
    // the CTA's own half of the two tiles, lanes 16-23 and 24-31 of the peer's (past the end: the last row's).
    // Four lookups in turn wait for the page table four times: 129 against 125 us for 36 trees of 51 nodes and 128 heads
    // after 2 keys, 24.6 against 23.8 for 4 of 8 nodes after 1,000 fp8 keys.
    auto find = [&](const TreeItem& t, int j, int& off) -> int {          // page and offset in it
      if (F8 && by_tma(t, t.tile + min(j + 1, t.n_tiles - 1))) return 0;  // then neither is fed
      const int half = rank ^ int(lane >> 4);
      const int pos = min((t.tile + j + int(lane >> 3 & 1)) * KT + half * 64 + r0 + int(lane & 7), t.ctx + t.n - 1);
      off = pos % p.lay.page;
      return p.lay.table[size_t(t.b) * p.lay.P + pos / p.lay.page];
    };
    // fp8: a lane holds 16 values of a row, two 16-byte columns of its atom's chunk.  Lanes of odd atoms take the rows of
    // a pair the other way round, so that a store's lanes meet all eight columns (row and column are xored) without
    // exchanging data (53.8 -> 53.0 us for 100,000 keys, 18.0 -> 17.7 for 8 trees of 20 after 30).  The instructions of
    // this expansion are what a fed fp8 tile waits for: converting one of the four words by integer instructions instead
    // takes 58.6 us, all four 70.4.
    const int sw = (lane >> 2) & 1, two = int(lane >> 4) ^ sw;
    const uint8_t* kv_k = p.kv + (lane + (lane >= 16 ? 1 : 0)) * 16;
    const uint8_t* kv_ks = p.kv + 256 + (lane >> 2);
    const uint8_t* kv_v = p.kv + (17 * rank + (lane & 15)) * 16;
    const uint8_t* kv_vs = p.kv + 256 + 4 * rank + ((lane & 15) >> 2);
    const uint32_t to_k = (lane >> 2) * CH + r0 * 128 + ((2 * (lane & 3)) << 4 ^ sw * 0x90);
    const uint32_t to_v = ((lane & 15) >> 2) * CH + r0 * 128 + ((2 * (lane & 3)) << 4 ^ two * 0x90);
    auto at = [&](int rows, int r) { return p.kv + int64_t(__shfl_sync(~0u, rows, r)) * RB; };
    TreeItem nx = p.work.items[i0];                     // items are read one ahead
    int off = 0, page = find(nx, 0, off), now = page * p.lay.page + off;
    pdl_wait();
    for (int i = i0; ok && i < i1; ++i) {
      const TreeItem it = nx;
      if (i + 1 < i1) nx = p.work.items[i + 1];
      const int end = it.ctx + it.n, nt = it.n_tiles;
      uint32_t odd = 0;                                 // this warp's rows with a NaN or an infinity, 8 bits per stage
      for (int j = 0; ok && j < nt; j += 2) {
        const int m = min(2, nt - j);
        // the next pair of tiles: this item's, or the next item's first
        const bool more = j + 2 < nt;
        const TreeItem& an = more ? it : nx;
        const int aj = more ? j + 2 : 0;
        const bool any = more || i + 1 < i1;
        // fp8: looked up here; bf16: after the first tile's keys, when the next item has been read (for 36 trees of 51
        // nodes x 128 heads after 2 keys 117.7 against 121.0 us; 100,000 fp8 keys take 55.4 that way and 53.4 this way)
        int next = 0;
        if (F8 && any) {
          page = find(an, aj, off);
          next = page * p.lay.page + off;
        }
        auto ahead = [&](int u) {                       // L2 prefetch two tiles on
          if (!any || aj + u >= an.n_tiles || by_tma(an, an.tile + aj + u)) return;
          const uint8_t* row = p.kv + int64_t(__shfl_sync(~0u, next, 8 * u + (lane >> 2))) * RB;
#pragma unroll
          for (int o = 0; o < RB; o += 512)
            if (o + int(lane & 3) * 128 < RB) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + o + (lane & 3) * 128));
        };
        for (int u = 0; ok && u < m; ++u) {
          const int s = (g + u) & 1, ph = ((g + u) >> 1) & 1, tile = it.tile + j + u;
          uint8_t* st = sK + s * STAGE;
          const bool fed = !by_tma(it, tile), tail = (tile + 1) * KT > it.ctx;
          if (fed) {
            const int rows = end - (tile * KT + rank * 64 + r0);        // rows of this warp that exist
            odd &= ~(0xFFu << (8 * s));
            if constexpr (F8) {
              uint4 pe[2];                                // RoPE pieces: lane = (row of four, piece)
              auto load_pe = [&]() {
  #pragma unroll
                for (int k = 0; k < 2; ++k)
                  if (NA == 9) pe[k] = reinterpret_cast<const uint4*>(at(now, 8 * u + 4 * k + (lane >> 3)))[33 + (lane & 7)];
              };
              auto store_pe = [&]() {
  #pragma unroll
                for (int k = 0; k < 2; ++k) {
                  if (NA != 9) break;
                  if (tail && 4 * k + int(lane >> 3) >= rows) pe[k] = zero;
                  put(st + 8 * CH, r0 + 4 * k + (lane >> 3), lane & 7, pe[k]);
                  if (tail) {
                    const uint32_t bad = __ballot_sync(~0u, odd16<F8>(pe[k]));
  #pragma unroll
                    for (int r = 0; r < 4; ++r)
                      if ((bad >> (8 * r)) & 0xFF) odd |= 1u << (8 * s + 4 * k + r);
                  }
                }
              };
              uint4 v[8];
              uint32_t sc[8];
#pragma unroll
              for (int r = 0; r < 8; ++r) {
                const int64_t o = int64_t(__shfl_sync(~0u, now, (8 * u + r) ^ sw)) * RB;
                v[r] = *reinterpret_cast<const uint4*>(kv_k + o);
                sc[r] = kv_ks[o];
              }
              load_pe();
              ok = wait(&pv0[s], ph ^ 1, kErrTimeoutEmpty) && wait(&pv1[s], ph ^ 1, kErrTimeoutEmpty);
#pragma unroll
              for (int r = 0; r < 8; ++r) {
                uint4 a, b;
                if (tail && (r ^ sw) >= rows) v[r] = zero;
                expand16(v[r], sc[r], a, b);
                *reinterpret_cast<uint4*>(st + (to_k ^ (r * 0x90))) = a;
                *reinterpret_cast<uint4*>(st + (to_k ^ (r * 0x90 ^ 0x10))) = b;
                if (tail) {
                  const uint32_t bad = __ballot_sync(~0u, odd16<F8>(a) || odd16<F8>(b));
                  if (bad & 0x0f0f0f0fu) odd |= 1u << (8 * s + r);
                  if (bad & 0xf0f0f0f0u) odd |= 1u << (8 * s + (r ^ 1));
                }
              }
              store_pe();
            } else {
              uint4 pe[2];
#pragma unroll
              for (int h = 0; h < 2; ++h) {             // four rows at a time; rows past the end are not read
                uint4 v[8];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  const uint4* src = reinterpret_cast<const uint4*>(at(now, 8 * u + 4 * h + r));
                  v[2 * r] = v[2 * r + 1] = zero;
                  if (4 * h + r < rows) { v[2 * r] = src[lane]; v[2 * r + 1] = src[32 + lane]; }
                }
                if (NA == 9) pe[h] = reinterpret_cast<const uint4*>(at(now, 8 * u + 4 * h + (lane >> 3)))[64 + (lane & 7)];
                if (h == 0) ok = wait(&pv0[s], ph ^ 1, kErrTimeoutEmpty) && wait(&pv1[s], ph ^ 1, kErrTimeoutEmpty);
                if (tail) {
#pragma unroll
                  for (int r = 0; r < 4; ++r) {
                    if (__any_sync(~0u, odd16<F8>(v[2 * r]) || odd16<F8>(v[2 * r + 1]))) odd |= 1u << (8 * s + 4 * h + r);
                  }
                  if (NA == 9) {
                    if (4 * h + int(lane >> 3) >= rows) pe[h] = zero;
                    const uint32_t bad = __ballot_sync(~0u, odd16<F8>(pe[h]));
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                      if ((bad >> (8 * r)) & 0xFF) odd |= 1u << (8 * s + 4 * h + r);
                  }
                }
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                  for (int k = 0; k < 2; ++k)
                    put(st + (k * 4 + (lane >> 3)) * CH, r0 + 4 * h + r, lane & 7, v[2 * r + k]);
                if (NA == 9) put(st + 8 * CH, r0 + 4 * h + (lane >> 3), lane & 7, pe[h]);
              }
            }
            fence_proxy_async();
          } else {
            ok = wait(&pv1[s], ph ^ 1, kErrTimeoutEmpty);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&kfull[s]), 0));
          if constexpr (F8) {
            if (fed) ahead(u);
          } else if (u == 0 && any) {
            page = find(an, aj, off);                   // not waited for before the second tile's keys
          }
        }
        if constexpr (!F8) {
          next = page * p.lay.page + off;
          for (int u = 0; u < m; ++u) ahead(u);
        }
        for (int u = 0; ok && u < m; ++u) {
          const int s = (g + u) & 1, ph = ((g + u) >> 1) & 1, tile = it.tile + j + u;
          uint8_t* st = sK + s * STAGE;
          if (!by_tma(it, tile)) {
            const bool tail = (tile + 1) * KT > it.ctx;
            const int rows = end - (tile * KT + (rank ^ 1) * 64 + r0);
            uint8_t* dst = st + (rank ? 0 : 4) * CH;
            if constexpr (F8) {
              uint4 v[4];                               // two rows per load: 16 lanes x 16 values
              uint32_t sc[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int64_t o = int64_t(__shfl_sync(~0u, now, 16 + 8 * u + 2 * k + two)) * RB;
                v[k] = *reinterpret_cast<const uint4*>(kv_v + o);
                sc[k] = kv_vs[o];
              }
              ok = wait(&sfull[s], ph, kErrTimeoutFull);
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                uint4 a, b;
                if (tail && 2 * k + two >= rows) v[k] = zero;
                expand16(v[k], sc[k], a, b);
                if (tail && odd16<F8>(a)) a = zero;
                if (tail && odd16<F8>(b)) b = zero;
                *reinterpret_cast<uint4*>(dst + (to_v ^ (k * 0x120))) = a;
                *reinterpret_cast<uint4*>(dst + (to_v ^ (k * 0x120 ^ 0x10))) = b;
              }
            } else {
              uint4 v[8];
#pragma unroll
              for (int r = 0; r < 8; ++r) v[r] = reinterpret_cast<const uint4*>(at(now, 16 + 8 * u + r))[32 * rank + lane];
              ok = wait(&sfull[s], ph, kErrTimeoutFull);
#pragma unroll
              for (int r = 0; r < 8; ++r) {
                if (tail && (r >= rows || odd16<F8>(v[r]))) v[r] = zero;
                put(dst + (lane >> 3) * CH, r0 + r, lane & 7, v[r]);
              }
            }
            // this CTA's own keys: rows that were marked lose their values
            for (uint32_t left = (odd >> (8 * s)) & 0xFF; left; left &= left - 1)
              put(st + (4 * rank + (lane >> 3)) * CH, r0 + __ffs(left) - 1, lane & 7, zero);
            fence_proxy_async();
          } else {
            ok = wait(&sfull[s], ph, kErrTimeoutFull);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&vfull[s]), 0));
        }
        g += m;
        now = next;
      }
      if (*abort_flag) ok = false;
    }
  } else {
    // ---------------- softmax, rescale, epilogue: lanes 0-63 / 64-127 hold the first / second 64 keys of the rows;
    // two warps share 32 lanes and take 32 score columns (and 128 of the 256 columns of O) each -------
    const int q = warp & 3, half = q >> 1, row = (q & 1) * 32 + int(lane), part = (int(warp) - 2 - FEED_WARPS) >> 2;
    const int me = part * 128 + q * 32 + int(lane);
    const uint32_t t_lane = tmem + (uint32_t(q * 32) << 16);
    auto mask_of = [&](const TreeItem& t) -> uint64_t {
      const int r = t.row * 128 + rank * 64 + row;
      return r < t.n * p.H ? uint64_t(p.mask[t.c0 + r / p.H]) : 0;
    };
    TreeItem nx = p.work.items[i0];                     // items and masks are read one ahead
    uint64_t next_mask = mask_of(nx);
    pdl_wait();
    int g = 0;
    bool ok = true;                       // after a failed wait the loop runs on without waiting: the block-level
    for (int i = i0; i < i1; ++i) {       // barriers below need all the warps
      const TreeItem it = nx;
      if (i + 1 < i1) nx = p.work.items[i + 1];
      const int ctx = it.ctx, c0 = it.c0, n = it.n;
      const int r = it.row * 128 + rank * 64 + row;
      const bool live = r < n * p.H;
      const int head = live ? r % p.H : 0;
      const uint64_t mask = next_mask;
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
          for (int c = part * 128; c < part * 128 + 128; c += 16) {
            uint32_t o[16];
            tmem_ld_32x32b_x16(t_lane + TM_O + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * keep);
            tmem_st_32x32b_x16(t_lane + TM_O + c, o);
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
      if (i + 1 < i1) next_mask = mask_of(nx);
      const int sl = (g - 1) & 1;
      ok = ok && wait(&pv1[sl], ((g - 1) >> 1) & 1, kErrTimeoutTmem);
      tc_fence_after();
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
      // O: a lane's row of 64 bf16 (32 fp32) columns at a time, transposed over four lanes, so that a store instruction
      // writes eight whole 128-byte lines instead of a sector of 32 (2.3 us of a one-tile call's 3.5 us epilogue)
      const int quad = (lane & 3) * 8, top = rank * 64 + (row & ~3);                // the four rows' first, in the tile
      const int rows_left = n * p.H - it.row * 128 - top;
      if (it.part < 0) {
        __nv_bfloat16* o = p.out + (size_t(c0) * p.H + it.row * 128 + top) * 512 + half * 256 + part * 128 + 2 * quad;
#pragma unroll 1
        for (int c = 0; c < 128; c += 64) {
          uint32_t v[32], x[32];
          tmem_ld_32x32b_x32(t_lane + TM_O + part * 128 + c, x);
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 16; ++k)
            v[k] = pack_bf16x2(__uint_as_float(x[2 * k]) * inv, __uint_as_float(x[2 * k + 1]) * inv);
          tmem_ld_32x32b_x32(t_lane + TM_O + part * 128 + c + 32, x);
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 16; ++k)
            v[16 + k] = pack_bf16x2(__uint_as_float(x[2 * k]) * inv, __uint_as_float(x[2 * k + 1]) * inv);
          quad_transpose(v, lane);
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (u < rows_left) store32(o + u * 512 + c, v + 8 * u);
        }
      } else {
        float* po = p.part_o + (size_t(it.part) * 128 + top) * 512 + half * 256 + part * 128 + quad;
#pragma unroll 1
        for (int c = 0; c < 128; c += 32) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(t_lane + TM_O + part * 128 + c, v);
          tmem_ld_wait();
          quad_transpose(v, lane);
#pragma unroll
          for (int u = 0; u < 4; ++u) store32(po + u * 512 + c, v + 8 * u);
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
// dims per thread, eight partial rows in flight with a running maximum.  With more than eight partial rows G groups of
// threads take every G-th one and are joined through shared memory (one row tile in 53 parts: 4 groups took a call of
// 20,000 keys from 20.8 to 18.1 us).
template <int G>
__global__ void __launch_bounds__(128 * G) tree_merge_kernel(const TreeMerge* __restrict__ merges, int H,
                                                             const float* __restrict__ part_o,
                                                             const float* __restrict__ part_ml,
                                                             const float* __restrict__ sink,
                                                             __nv_bfloat16* __restrict__ out) {
  const TreeMerge mg = merges[blockIdx.x];              // made by the host
  pdl_entry();
  const int row = blockIdx.y, r = mg.row * 128 + row, group = threadIdx.x >> 7, dim = threadIdx.x & 127;
  if (r >= mg.rows) return;
  const float2* ml = reinterpret_cast<const float2*>(part_ml) + size_t(mg.part) * 128 + row;
  const float4* po = reinterpret_cast<const float4*>(part_o) + (size_t(mg.part) * 128 + row) * 128 + dim;
  float M = sink ? sink[r % H] * 1.4426950408889634f : -INFINITY;
  float L = sink && group == 0 ? 1.f : 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = group; s0 < mg.n; s0 += 8 * G) {
    float2 v[8];
    float4 o[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const int at = s0 + s * G;
      v[s] = at < mg.n ? ml[at * 128] : make_float2(-INFINITY, 0.f);
      o[s] = at < mg.n ? po[size_t(at) * 128 * 128] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float top = M;
#pragma unroll
    for (int s = 0; s < 8; ++s) top = fmaxf(top, v[s].x);
    const float ref = top == -INFINITY ? 0.f : top, keep = exp2f(M - ref);
    acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
    L *= keep;
    M = top;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const float w = exp2f(v[s].x - ref);
      L += w * v[s].y;
      acc.x += w * o[s].x; acc.y += w * o[s].y; acc.z += w * o[s].z; acc.w += w * o[s].w;
    }
  }
  if constexpr (G > 1) {
    __shared__ float4 s_acc[G][128];
    __shared__ float2 s_ml[G];
    s_acc[group][dim] = acc;
    if (dim == 0) s_ml[group] = make_float2(M, L);
    __syncthreads();
    if (group) return;
    float top = M;
#pragma unroll
    for (int k = 1; k < G; ++k) top = fmaxf(top, s_ml[k].x);
    const float ref = top == -INFINITY ? 0.f : top;
    const float keep = exp2f(M - ref);
    acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
    L *= keep;
#pragma unroll
    for (int k = 1; k < G; ++k) {
      const float w = exp2f(s_ml[k].x - ref);
      const float4 o = s_acc[k][dim];
      L += w * s_ml[k].y;
      acc.x += w * o.x; acc.y += w * o.y; acc.z += w * o.z; acc.w += w * o.w;
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  reinterpret_cast<uint2*>(out + (size_t(mg.c0) * H + r) * 512)[dim] =
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

cudaError_t tree_mla(const void* q, int T, int H, int D, bool f8, const void* kv, int64_t S, const TreeLayout& lay,
                     const TreeWork& work, const int64_t* mask, float scale, const float* sink, float* part_o,
                     float* part_ml, void* staged, int* status, void* out, cudaStream_t s) {
  using namespace tree;
  if (!encode_fn()) return cudaErrorNotSupported;
  if (D != 576 && D != 512) return cudaErrorInvalidValue;
  const int how = staged ? STAGED : f8 || lay.page % 64 != 0 ? FEED : PAGED;
  cudaError_t e;
  Maps m;
  if (!row_map(&m.q, f8, q, int64_t(T) * H, D, 64, D / 64)) return cudaErrorInvalidValue;
  m.kv4 = m.kv1 = m.q;
  const void* rows = staged ? staged : kv;
  const int64_t n_rows = staged ? int64_t(work.n_stage) * KT : S;
  if (how != FEED && !(row_map(&m.kv4, f8, rows, n_rows, D, 64, 4) && row_map(&m.kv1, f8, rows, n_rows, D, 64, 1)))
    return cudaErrorInvalidValue;
  if (staged &&
      (e = launch_k(f8 ? tree_stage_kernel<true> : tree_stage_kernel<false>, dim3(work.n_stage * 4), 256, 0, s,
                    reinterpret_cast<const uint8_t*>(kv), lay, work.stage, D, reinterpret_cast<uint16_t*>(staged))) !=
          cudaSuccess)
    return e;
  Params p;
  p.lay = lay; p.work = work; p.mask = mask;
  p.kv = reinterpret_cast<const uint8_t*>(kv);
  p.H = H; p.how = how;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.sink = sink; p.part_o = part_o; p.part_ml = part_ml; p.status = status;
  p.out = reinterpret_cast<__nv_bfloat16*>(out);
  Kernel f = D == 576 ? (f8 ? tree_mla_kernel<9, true> : tree_mla_kernel<9, false>)
                      : (f8 ? tree_mla_kernel<8, true> : tree_mla_kernel<8, false>);
  if ((e = smem_optin(f, SMEM)) != cudaSuccess) return e;
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = pair_config(work.clusters, attr, s);
  if ((e = cudaLaunchKernelEx(&cfg, f, m, p)) != cudaSuccess || !work.n_merges) return e;
  const bool many = work.most_parts > 8;
  return launch_k(many ? tree_merge_kernel<4> : tree_merge_kernel<1>, dim3(work.n_merges, 128), many ? 512 : 128, 0, s,
                  work.merges, H, part_o, part_ml, sink, p.out);
}

}  // namespace cb
