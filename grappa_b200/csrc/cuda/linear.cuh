// Linear layer with everything that follows it in the epilogue:
//
//   z = A W^T + bias            bf16 operands, fp32 accumulation in tensor memory
//   out = dropout(act(z)) + residual,   z kept as bf16 rows or in 8 bits
//
// The CTAs walk the 128 x BN output tiles:
//   warp 0      TMA producer of the A and W tiles of each 64-wide k-block (a ring of
//               128B-swizzled buffers that runs across tiles)
//   warp 1      issues tcgen05.mma (M = 128, N = BN, K = 16) into one of two TMEM
//               accumulators, so the epilogue of a tile overlaps the products of the next.
//               256-column tiles are made by CTA pairs (cta_group::2, M = 256): each CTA
//               loads half of W's tile, which halves what the products read of it
//   warps 2..   epilogue: each warp owns 32 rows (a TMEM lane quarter) x 64 columns, in two
//               halves.  A half's residual comes by TMA into the very buffer that the
//               output leaves from (a lane adds and overwrites its own 16-byte pieces), and
//               while one half is computed the other's store leaves and its next residual
//               comes.
//
// At the widths of graph layers (K and N of a few hundred) the kernel is bound by HBM:
// A, residual, out and the kept z are each moved once.  A 32-column group of the 8-bit
// form is 32 accumulator registers of one thread, so its largest magnitude needs no
// exchange.
//
// The tensor core adds each 16 columns of K into its fp32 accumulator by truncation: z is off by
// up to K / 16 steps of 2^-23 of the largest partial sum, far below bf16's or a code's step,
// but a value that close to the middle between two codes may get the other one.
//
// Measured: 139058 x 512 x 256 39 us (SiLU, residual and 8-bit z: 59, 85 % of the copy's
// rate), 131072 x 1024 x 1024 195 us = 1410 TFLOP/s (263).
//
// Rows >= the live count are not written.  Barrier waits are bounded as in gemm.cu.
#pragma once
#include <algorithm>

#include "ckpt8.cuh"
#include "grappa/rng.h"
#include "kernels.h"
#include "linear_act.cuh"
#include "tcgen05.cuh"

namespace grappa {
namespace dev {

namespace {

constexpr int BM = 128;
constexpr int BK = 64;

// A warp of the epilogue owns 32 rows x 64 columns of the tile, in two half panels of output /
// residual.  The 256-wide tile takes a whole SM (16 epilogue warps);
// narrower tiles share it (2 and 3 CTAs), so that as many warps work on epilogues.  What the
// epilogue needs no room for (RES: residuals, Q8: codes) goes to the ring: a load takes some
// 2000 cycles under load, a stage's products 640 (131072 x 1024 x 1024: 263 / 224 / 215 us
// with 3 / 4 / 5 stages).  With codes, though, a second half panel is worth more than a fifth
// stage unless the products are long (139058 x 208 x 256 with GELU 39.4 / 41.5 us, 65536 x
// 1024 x 512 74 / 71).
template <int BN, int CG, bool RES, bool Q8>
struct LSmem {
  static constexpr int kEpi = BN / 16;                       // epilogue warps
  static constexpr int kCtas = BN == 256 ? 1 : (BN == 128 ? 2 : 3);
  static constexpr int kThreads = 64 + 32 * kEpi;
  static constexpr int kABytes = BM * BK * 2;
  static constexpr int kBRows = BN / CG;                     // a pair of CTAs shares W's tile
  static constexpr int kBBytes = kBRows * BK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kPanels = CG == 2 && !RES && !Q8 ? 1 : 2;  // of 32 x 32 bf16 a warp
  static constexpr int kOutBytes = kEpi * kPanels * 2048;
  static constexpr bool kCodePanel = CG == 2 && Q8;          // and a 32 x 64 panel of codes
  static constexpr int kCodeBytes = kCodePanel ? kEpi * 2048 : 0;
  static constexpr int kBudget = 226 * 1024 / kCtas - 2048 - kOutBytes - kCodeBytes;
  static constexpr int kMost = CG == 2 ? 6 : 4;
  static constexpr int kStages = kBudget / kStageBytes > kMost ? kMost : kBudget / kStageBytes;
  static constexpr int kTmemCols = 2 * BN;
  static constexpr int kBytes = kStages * kStageBytes + kOutBytes + kCodeBytes + 1024 /*align*/;
  static_assert(kStages >= 2 && kCtas * (kBytes + 512) <= 227 * 1024 && kCtas * kTmemCols <= 512, "linear: resources");
};

// keeps the sign of what a ReLU reads: a positive value's code is at least 1
__device__ __forceinline__ uint2 codes8_relu(const float* v, float inv) {
  uint2 q = codes8(v, inv);
  if (inv == 0.f) return q;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (v[i] > 0.f && ((q.x >> (8 * i)) & 0xFFu) == 0u) q.x |= 1u << (8 * i);
    if (v[4 + i] > 0.f && ((q.y >> (8 * i)) & 0xFFu) == 0u) q.y |= 1u << (8 * i);
  }
  return q;
}

template <int BN, int CG, int ACT, bool RES, bool Q8, bool ANY>
__global__ void __launch_bounds__(LSmem<BN, CG, true, true>::kThreads, LSmem<BN, CG, true, true>::kCtas)
    linear_fwd_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                      const __grid_constant__ CUtensorMap tmR, const __grid_constant__ CUtensorMap tmO,
                      const __grid_constant__ CUtensorMap tmQ, LinearArgs a) {
  using S = LSmem<BN, CG, RES || ANY, Q8 || ANY>;
  constexpr int kStages = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full_bar[kStages], empty_bar[kStages], acc_full[2], acc_empty[2], res_full[S::kEpi][2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;

  // what the epilogue does: template parameters of the usual combinations, so that the 32
  // values of a thread meet no branches.  ANY reads all of it from the arguments and has dropout
  // and z in bf16: 69529 x 256 x 256 with ReLU executes 190 instructions a warp and 32 columns
  // (all warps counted), by ANY with z in bf16 586, by ANY with dropout 877
  const int act = ANY ? a.act : ACT;
  const bool has_res = ANY ? a.residual != nullptr : RES;
  const bool has_q8 = ANY ? a.q8.q != nullptr : Q8;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* out_area = smem + kStages * S::kStageBytes;
  uint8_t* code_area = out_area + S::kOutBytes;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], CG * S::kEpi);
      for (int w = 0; w < S::kEpi; ++w) mbar_init(&res_full[w][b], 1);
    }
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_map(&tmA);
    prefetch_map(&tmW);
    prefetch_map(&tmO);
    if (has_res) prefetch_map(&tmR);
  }
  if (warp == 1) CG == 2 ? tmem_alloc_pair(&tmem_slot, S::kTmemCols) : tmem_alloc(&tmem_slot, S::kTmemCols);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();  // both CTAs' barriers are ready
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = tmem_slot;
  // all of this may run while the kernel before is ending; its results are read from here on
  GB_PDL_ENTRY();
  const int M = live_rows(a.n_ptr, a.cap);
  const int kbs = (a.K + BK - 1) / BK;
  const int n_tiles = (a.N + BN - 1) / BN;
  // a tile is CG * 128 rows x BN columns; CTA `rank` of the pair has rows rank * 128 .. + 127
  constexpr int kTileM = BM * CG;
  const int64_t tiles = static_cast<int64_t>((M + kTileM - 1) / kTileM) * n_tiles;
  const int64_t first = blockIdx.x / CG, step = gridDim.x / CG;
  const int rank = CG == 2 ? static_cast<int>(cluster_rank()) : 0;

  // the two issuing warps stay converged; one elected lane issues (elect_one)
  if (warp == 0) {
    uint32_t it = 0;
    bool stop = false;
    for (int64_t t = first; t < tiles && !stop; t += step) {
      const int m0 = static_cast<int>(t / n_tiles) * kTileM + rank * BM;
      const int n0 = static_cast<int>(t % n_tiles) * BN + rank * S::kBRows;
      for (int kb = 0; kb < kbs; ++kb, ++it) {
        const int s = static_cast<int>(it % kStages);
        if (it >= static_cast<uint32_t>(kStages) &&
            !mbar_wait_all(&empty_bar[s], ((it / kStages) & 1u) ^ 1u, &abort_flag)) {
          if (lane == 0) set_error(a.err, kErrMmaTimeout);
          abort_flag = 1;
          stop = true;
          break;
        }
        uint8_t* sa = smem + s * S::kStageBytes;
        if (elect_one()) {
          if constexpr (CG == 2) {
            // both CTAs' loads complete on the issuing CTA's barrier
            if (rank == 0) mbar_expect_tx(&full_bar[s], 2 * S::kStageBytes);
            const uint32_t bar = cluster_addr(&full_bar[s], 0);
            tma_load_2d_pair(sa, &tmA, bar, kb * BK, m0);
            tma_load_2d_pair(sa + S::kABytes, &tmW, bar, kb * BK, n0);
          } else {
            mbar_expect_tx(&full_bar[s], S::kStageBytes);
            tma_load_2d(sa, &tmA, &full_bar[s], kb * BK, m0);
            tma_load_2d(sa + S::kABytes, &tmW, &full_bar[s], kb * BK, n0);
          }
        }
        __syncwarp();
      }
    }
    // on abort, wait (bounded) for the loads still in flight (of both CTAs)
    if (abort_flag && rank == 0) {
      for (uint32_t i = it > static_cast<uint32_t>(kStages) ? it - kStages : 0u; i < it; ++i) {
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(&full_bar[i % kStages], (i / kStages) & 1u) && globaltimer_ns() - t0 < kWaitNs) {
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      constexpr uint32_t idesc = umma_idesc(kTileM, BN, false, false);
      uint32_t it = 0;
      int lt = 0;
      bool stop = false;
      for (int64_t t = first; t < tiles && !stop; t += step, ++lt) {
        const int b = lt & 1;
        const uint32_t last = ((lt >> 1) - 1) & 1u;
        if (lt >= 2 && !(CG == 2 ? mbar_wait_cluster(&acc_empty[b], last, &abort_flag)
                                 : mbar_wait_all(&acc_empty[b], last, &abort_flag))) {
          if (lane == 0) set_error(a.err, kErrMmaTimeout);
          abort_flag = 1;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t d = tmem_base + static_cast<uint32_t>(b * BN);
        for (int kb = 0; kb < kbs; ++kb, ++it) {
          const int s = static_cast<int>(it % kStages);
          if (!mbar_wait_all(&full_bar[s], (it / kStages) & 1u, &abort_flag)) {
            if (lane == 0) set_error(a.err, kErrMmaTimeout);
            abort_flag = 1;
            stop = true;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t sa = smem_u32(smem + s * S::kStageBytes);
          const uint32_t sb = sa + S::kABytes;
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < BK / 16; ++kk) {
              const uint32_t acc = (kb > 0 || kk > 0) ? 1u : 0u;
              const uint64_t da = umma_desc(sa + kk * 32, 16, 1024), db = umma_desc(sb + kk * 32, 16, 1024);
              CG == 2 ? umma_f16_pair(d, da, db, idesc, acc) : umma_f16(d, da, db, idesc, acc);
            }
            CG == 2 ? umma_commit_pair(&empty_bar[s]) : umma_commit(&empty_bar[s]);
            if (kb == kbs - 1) CG == 2 ? umma_commit_pair(&acc_full[b]) : umma_commit(&acc_full[b]);
          }
          __syncwarp();
        }
      }
    }
  } else {
    const int w = warp - 2;
    const int quarter = warp & 3;  // TMEM lanes that this warp may read
    const int col0 = (w / 4) * 64;
    uint8_t* panels = out_area + w * (S::kPanels * 2048);  // of 32 rows x 32 columns
    uint8_t* codes = code_area + w * 2048;
    const uint64_t key = ANY && a.dropout_p > 0.f ? hop_key(static_cast<uint64_t>(a.counters[0]) ^ 0xD80Full,
                                                            static_cast<uint64_t>(a.counters[1]),
                                                            static_cast<uint64_t>(a.counters[2]), a.dropout_salt)
                                                  : 0ull;
    const uint32_t thr8 = dropout_thr8(a.dropout_p);
    const float keep_scale = dropout_scale8(thr8);
    // two exponent bytes of a row at an even address
    const bool e_pairs = ((reinterpret_cast<uintptr_t>(a.q8.e) | static_cast<uintptr_t>(a.q8.lde)) & 1u) == 0;
    const bool bias16 = (reinterpret_cast<uintptr_t>(a.bias) & 15u) == 0;
    const int n_pad = (a.N + 7) / 8 * 8;
    const int n_code = (a.N + 31) / 32 * 32;
    // the lane's 16-byte pieces of a 64-byte row, 64B-swizzled (panels and codes)
    const int swz = (lane >> 1) & 3;
    auto ask = [&](int64_t t, int h) {  // lane 0: half h of tile t's residual panel
      mbar_expect_tx(&res_full[w][h], 2048);
      tma_load_2d(panels + h * 2048, &tmR, &res_full[w][h], static_cast<int>(t % n_tiles) * BN + col0 + h * 32,
                  static_cast<int>(t / n_tiles) * kTileM + rank * BM + quarter * 32);
    };
    if (has_res && lane == 0 && first < tiles) ask(first, 0);
    int asked = first < tiles ? 1 : 0, taken = 0;  // residual half panels asked for and arrived
    int lt = 0;
    bool stop = false;
    for (int64_t t = first; t < tiles && !stop; t += step, ++lt) {
      const int m0 = static_cast<int>(t / n_tiles) * kTileM + rank * BM + quarter * 32;
      const int nc0 = static_cast<int>(t % n_tiles) * BN + col0;
      const int m = m0 + lane;
      const bool live = m < M;
      const bool slab_full = m0 + 32 <= M;  // rows past M are not written: no TMA store of such a slab
      const int ab = lt & 1;
      if (!mbar_wait_all(&acc_full[ab], (lt >> 1) & 1u, &abort_flag)) {
        if (lane == 0) set_error(a.err, kErrMmaTimeout);
        abort_flag = 1;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t trow =
          tmem_base + static_cast<uint32_t>(ab * BN + col0) + (static_cast<uint32_t>(quarter * 32) << 16);
      uint32_t bytes = 0;  // exponents of the two halves
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        const int nc = nc0 + h * 32;
        const bool whole = nc + 32 <= a.N;
        const bool code_cols = nc < n_code;
        uint8_t* panel = panels + (S::kPanels == 2 ? h * 2048 : 0);
        float v[32];
        tmem_ld32(trow + h * 32, v);
        if (lane == 0) {
          // what is written below has left: this half's panel, two stores ago (a store ago, where
          // there is one panel); with a residual the other half's panel too, into which the next
          // residual comes while this one is used; the code panel, a store ago
          if (has_res || S::kPanels == 1 || (S::kCodePanel && has_q8 && h == 0)) {
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            if (has_res && h == 0) ask(t, 1);
            if (has_res && h == 1 && t + step < tiles) ask(t + step, 0);
          } else {
            asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
          }
        }
        if (h == 0 || t + step < tiles) ++asked;
        __syncwarp();
        if (has_res) {
          if (!mbar_wait_all(&res_full[w][h], lt & 1u, &abort_flag)) {
            if (lane == 0) set_error(a.err, kErrMmaTimeout);
            abort_flag = 1;
            stop = true;
            break;
          }
          ++taken;
        }
        if (whole && bias16) {
          if (a.bias) {
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const float4 b = __ldg(reinterpret_cast<const float4*>(a.bias + nc + j));
              unpack(add2(f2(v[j], v[j + 1]), f2(b.x, b.y)), v[j], v[j + 1]);
              unpack(add2(f2(v[j + 2], v[j + 3]), f2(b.z, b.w)), v[j + 2], v[j + 3]);
            }
          }
        } else if (a.bias) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] += nc + j < a.N ? __ldg(a.bias + nc + j) : 0.f;
        }
        if (ANY && a.z && live && nc < a.N) {
          __nv_bfloat16* dst = a.z + static_cast<int64_t>(m) * a.ldz + nc;
#pragma unroll
          for (int j = 0; j < 32; j += 8)
            if (nc + j < n_pad) *reinterpret_cast<uint4*>(dst + j) = f32_to_bf16x8(v + j);
        }
        uint32_t c[8];
        float inv = 0.f;
        uint32_t byte = 0;
        if (has_q8) {
          byte = group8_byte(max_nan(abs_max3(abs_max8(v), abs_max8(v + 8), abs_max8(v + 16)), abs_max8(v + 24)));
          inv = group8_inv(byte);
          bytes |= byte << (8 * h);
        }
        uint32_t keep = 0xFFFFFFFFu;
        if (ANY && a.dropout_p > 0.f)
          keep = dropout_keep_bits(key, static_cast<uint64_t>(m) * static_cast<uint64_t>(a.ldo) + static_cast<uint64_t>(nc),
                                   32, thr8);
        // eight columns at a time: codes, activation, residual, the piece of the panel
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float* x = v + 8 * q;
          if (has_q8) {
            const uint2 cu = act == kActRelu ? codes8_relu(x, inv) : codes8(x, inv);
            c[2 * q] = cu.x, c[2 * q + 1] = cu.y;
          }
          if (act == kActRelu) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = max_nan(x[j], 0.f);
          } else if (act == kActGelu) {
#pragma unroll
            for (int j = 0; j < 8; j += 2) gelu2(x + j);
          } else if (act == kActSilu) {
#pragma unroll
            for (int j = 0; j < 8; j += 2) silu2(x + j);
          }
          if (ANY && a.dropout_p > 0.f) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = (keep >> (8 * q + j)) & 1u ? x[j] * keep_scale : 0.f;
          }
          uint4* piece = reinterpret_cast<uint4*>(panel + lane * 64 + ((q ^ swz) << 4));
          if (has_res) {
            float r[8];
            bf16x8_to_f32(*piece, r);
#pragma unroll
            for (int j = 0; j < 8; j += 2) unpack(add2(f2(x[j], x[j + 1]), f2(r[j], r[j + 1])), x[j], x[j + 1]);
          }
          uint4 o = f32_to_bf16x8(x);
          if (has_res && !whole) o = first_columns(o, a.N - nc - 8 * q);  // the residual's pad columns
          *piece = o;
        }
        if (has_q8) {
          if (live && code_cols) {
            uint8_t* e = a.q8.e + static_cast<int64_t>(m) * a.q8.lde + (nc >> 5);
            if (!e_pairs || nc0 + 32 >= n_code)
              *e = static_cast<uint8_t>(byte);
            else if (h == 1)
              *reinterpret_cast<uint16_t*>(e - 1) = static_cast<uint16_t>(bytes);
          }
          if constexpr (S::kCodePanel) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
              *reinterpret_cast<uint4*>(codes + lane * 64 + (((h * 2 + u) ^ swz) << 4)) =
                  make_uint4(c[4 * u], c[4 * u + 1], c[4 * u + 2], c[4 * u + 3]);
          }
          if ((!S::kCodePanel || !slab_full) && code_cols) {
            // neighbouring lanes trade halves, so that a store writes whole 32-byte sectors:
            // first the even lane's row (16 bytes by each), then the odd lane's
            const bool odd = lane & 1;
            uint32_t got[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) got[u] = __shfl_xor_sync(0xffffffffu, odd ? c[u] : c[4 + u], 1);
            const uint4 one = odd ? make_uint4(got[0], got[1], got[2], got[3]) : make_uint4(c[0], c[1], c[2], c[3]);
            const uint4 two = odd ? make_uint4(c[4], c[5], c[6], c[7]) : make_uint4(got[0], got[1], got[2], got[3]);
            const int me = m - (lane & 1);
            int8_t* dst = a.q8.q + static_cast<int64_t>(me) * a.q8.ldq + nc + (odd ? 16 : 0);
            if (me < M) *reinterpret_cast<uint4*>(dst) = one;
            if (me + 1 < M) *reinterpret_cast<uint4*>(dst + a.q8.ldq) = two;
          }
        }
        if (!slab_full && live) {
          // a slab that crosses the last live row: its rows by plain stores
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (nc + 8 * q < n_pad)
              *reinterpret_cast<uint4*>(a.out + static_cast<int64_t>(m) * a.ldo + nc + 8 * q) =
                  *reinterpret_cast<const uint4*>(panel + lane * 64 + ((q ^ swz) << 4));
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          if (slab_full && nc < a.N) tma_store_2d(&tmO, panel, nc, m0);
          if (S::kCodePanel && has_q8 && h == 1 && slab_full && nc0 < a.N) tma_store_2d(&tmQ, codes, nc0, m0);
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
      }
      // the accumulator is read: the products of the tile after the next may start
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) CG == 2 ? mbar_arrive_cluster(cluster_addr(&acc_empty[ab], 0)) : mbar_arrive(&acc_empty[ab]);
    }
    if (lane == 0) {
      // the panels are in shared memory that ends with the CTA: wait for the stores'
      // reads, and after an abort (bounded) for residual panels still on their way
      asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      if (abort_flag && has_res) {
        for (int k = taken; k < asked; ++k) {
          const uint64_t t0 = globaltimer_ns();
          while (!mbar_try_wait(&res_full[w][k & 1], (k >> 1) & 1u) && globaltimer_ns() - t0 < kWaitNs) {
          }
        }
      }
    }
  }
  __syncthreads();
  // neither CTA leaves while the other may still arrive on its barriers or read its memory
  if constexpr (CG == 2) cluster_sync();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    CG == 2 ? tmem_dealloc_pair(tmem_base, S::kTmemCols) : tmem_dealloc(tmem_base, S::kTmemCols);
  }
}

template <int BN, int CG, int ACT, bool RES, bool Q8, bool ANY>
void linear_kernel(const LinearArgs& a, cudaStream_t stream) {
  using S = LSmem<BN, CG, RES || ANY, Q8 || ANY>;
  const int64_t n_pad = ceil_div(a.N, 8) * 8;
  const CUtensorMap ma = tensor_map_bf16(a.A, a.a_rows, a.K, a.lda, BM);
  const CUtensorMap mw = tensor_map_bf16(a.W, a.N, a.K, a.ldw, S::kBRows);
  const CUtensorMap mo = tensor_map_2d(CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.out, a.out_rows, n_pad, a.ldo, 32, 32,
                                       CU_TENSOR_MAP_SWIZZLE_64B);
  const CUtensorMap mr = a.residual ? tensor_map_2d(CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.residual, a.r_rows, n_pad,
                                                    a.ldr, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B)
                                    : mo;
  const CUtensorMap mq = S::kCodePanel && a.q8.q
                             ? tensor_map_u8(a.q8.q, a.q_rows, ceil_div(a.N, 32) * 32, a.q8.ldq, 64, 32,
                                             CU_TENSOR_MAP_SWIZZLE_64B)
                             : mo;
  auto kern = linear_fwd_kernel<BN, CG, ACT, RES, Q8, ANY>;
  set_smem(reinterpret_cast<const void*>(kern), S::kBytes);
  const int64_t tiles = ceil_div(a.cap, BM * CG) * ceil_div(a.N, BN);
  launch_cluster_k(kern, dim3(static_cast<unsigned>(std::min<int64_t>(tiles, sm_count() * S::kCtas / CG) * CG)),
                   dim3(S::kThreads), CG, S::kBytes, stream, ma, mw, mr, mo, mq, a);
  GB_LAUNCH_CHECK();
}

// the kernel of a tile shape for what the epilogue has to do
template <int BN, int CG>
void linear_tiles(const LinearArgs& a, cudaStream_t stream) {
  if (a.z || a.dropout_p > 0.f) return linear_kernel<BN, CG, 0, false, false, true>(a, stream);
#define GB_LINEAR_ACT(ACT)                                                                              \
  if (a.act == ACT) {                                                                                   \
    if (a.residual)                                                                                     \
      return a.q8.q ? linear_kernel<BN, CG, ACT, true, true, false>(a, stream)                          \
                    : linear_kernel<BN, CG, ACT, true, false, false>(a, stream);                        \
    return a.q8.q ? linear_kernel<BN, CG, ACT, false, true, false>(a, stream)                           \
                  : linear_kernel<BN, CG, ACT, false, false, false>(a, stream);                         \
  }
  GB_LINEAR_ACT(kActNone)
  GB_LINEAR_ACT(kActRelu)
  GB_LINEAR_ACT(kActGelu)
  GB_LINEAR_ACT(kActSilu)
#undef GB_LINEAR_ACT
}

}  // namespace

}  // namespace dev
}  // namespace grappa
