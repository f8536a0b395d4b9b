// Linear layer with everything that follows it in the epilogue:
//
//   z = A W^T + bias            bf16 operands, fp32 accumulation in tensor memory
//   out = dropout(act(z)) + residual,   z kept as bf16 rows or in 8 bits
//
// One CTA per SM walks the 128 x BN output tiles:
//   warp 0      TMA producer of the A and W tiles of each 64-wide k-block (a ring of
//               128B-swizzled buffers that runs across tiles)
//   warp 1      issues tcgen05.mma (M = 128, N = BN, K = 16) into one of two TMEM
//               accumulators, so the epilogue of a tile overlaps the products of the next
//   warps 2..   epilogue: each warp owns 32 rows (a TMEM lane quarter) and the tile's
//               columns in panels of 64.  The residual's panel comes by TMA into the very
//               buffer that the output panel leaves from (a lane adds and overwrites its
//               own 16-byte pieces), two panels a warp: while one is computed, the other's
//               store drains and the next residual panel loads.
//
// At the widths of graph layers (K and N of a few hundred) the kernel is bound by HBM:
// A, residual, out and the kept z are each moved once.  A 32-column group of the 8-bit
// form is 32 accumulator registers of one thread, so its largest magnitude needs no
// exchange.
//
// Rows >= the live count are not written.  Barrier waits are bounded as in gemm.cu.
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

template <int BN>
struct LSmem {
  static constexpr int kEpi = BN >= 128 ? 8 : 4;             // epilogue warps
  static constexpr int kCols = BN / (kEpi / 4);              // columns of a warp
  static constexpr int kPanels = kCols / 64;
  static constexpr int kThreads = 64 + 32 * kEpi;
  static constexpr int kABytes = BM * BK * 2;
  static constexpr int kBBytes = BN * BK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kOutBytes = kEpi * 2 * 4096;          // two 32 x 64 bf16 panels a warp
  static constexpr int kCodeBytes = kEpi * 2048;             // one 32 x 64 code panel a warp
  static constexpr int kBudget = 226 * 1024 - kOutBytes - kCodeBytes;
  static constexpr int kStages = kBudget / kStageBytes > 8 ? 8 : kBudget / kStageBytes;
  static constexpr int kTmemCols = 2 * BN;
  static constexpr int kBytes = kStages * kStageBytes + kOutBytes + kCodeBytes + 1024 /*align*/;
  static_assert(kStages >= 3 && kBytes <= 226 * 1024, "linear: shared memory");
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

template <int BN>
__global__ void __launch_bounds__(LSmem<BN>::kThreads, 1)
    linear_fwd_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                      const __grid_constant__ CUtensorMap tmR, const __grid_constant__ CUtensorMap tmO,
                      const __grid_constant__ CUtensorMap tmQ, LinearArgs a) {
  GB_PDL_ENTRY();
  using S = LSmem<BN>;
  constexpr int kStages = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full_bar[kStages], empty_bar[kStages], acc_full[2], acc_empty[2], res_full[S::kEpi][2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;

  const int M = live_rows(a.n_ptr, a.cap);
  const int kbs = (a.K + BK - 1) / BK;
  const int n_tiles = (a.N + BN - 1) / BN;
  const int64_t tiles = static_cast<int64_t>((M + BM - 1) / BM) * n_tiles;
  if (static_cast<int64_t>(blockIdx.x) >= tiles) return;

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
      mbar_init(&acc_empty[b], S::kEpi);
      for (int w = 0; w < S::kEpi; ++w) mbar_init(&res_full[w][b], 1);
    }
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(&tmem_slot, S::kTmemCols);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;
      bool stop = false;
      for (int64_t t = blockIdx.x; t < tiles && !stop; t += gridDim.x) {
        const int m0 = static_cast<int>(t / n_tiles) * BM, n0 = static_cast<int>(t % n_tiles) * BN;
        for (int kb = 0; kb < kbs; ++kb, ++it) {
          const int s = static_cast<int>(it % kStages);
          if (it >= static_cast<uint32_t>(kStages) &&
              !mbar_wait(&empty_bar[s], ((it / kStages) & 1u) ^ 1u, &abort_flag)) {
            set_error(a.err, kErrMmaTimeout);
            abort_flag = 1;
            stop = true;
            break;
          }
          uint8_t* sa = smem + s * S::kStageBytes;
          mbar_expect_tx(&full_bar[s], S::kStageBytes);
          tma_load_2d(sa, &tmA, &full_bar[s], kb * BK, m0);
          tma_load_2d(sa + S::kABytes, &tmW, &full_bar[s], kb * BK, n0);
        }
      }
      // on abort, wait (bounded) for the loads still in flight
      if (abort_flag) {
        for (uint32_t i = it > static_cast<uint32_t>(kStages) ? it - kStages : 0u; i < it; ++i) {
          const uint64_t t0 = globaltimer_ns();
          while (!mbar_try_wait(&full_bar[i % kStages], (i / kStages) & 1u) && globaltimer_ns() - t0 < kWaitNs) {
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = umma_idesc(BM, BN, false, false);
      uint32_t it = 0;
      int lt = 0;
      bool stop = false;
      for (int64_t t = blockIdx.x; t < tiles && !stop; t += gridDim.x, ++lt) {
        const int b = lt & 1;
        if (lt >= 2 && !mbar_wait(&acc_empty[b], ((lt >> 1) - 1) & 1u, &abort_flag)) {
          set_error(a.err, kErrMmaTimeout);
          abort_flag = 1;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        for (int kb = 0; kb < kbs; ++kb, ++it) {
          const int s = static_cast<int>(it % kStages);
          if (!mbar_wait(&full_bar[s], (it / kStages) & 1u, &abort_flag)) {
            set_error(a.err, kErrMmaTimeout);
            abort_flag = 1;
            stop = true;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t sa = smem_u32(smem + s * S::kStageBytes);
          const uint32_t sb = sa + S::kABytes;
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk)
            umma_f16(tmem_base + static_cast<uint32_t>(b * BN), umma_desc(sa + kk * 32, 16, 1024),
                     umma_desc(sb + kk * 32, 16, 1024), idesc, (kb > 0 || kk > 0) ? 1u : 0u);
          umma_commit(&empty_bar[s]);
        }
        if (!stop) umma_commit(&acc_full[b]);
      }
    }
  } else {
    const int w = warp - 2;
    const int quarter = warp & 3;  // TMEM lanes that this warp may read
    const int col0 = (w / 4) * S::kCols;
    uint8_t* panel[2] = {out_area + w * 8192, out_area + w * 8192 + 4096};
    uint8_t* codes = code_area + w * 2048;
    const uint64_t key = a.dropout_p > 0.f ? hop_key(static_cast<uint64_t>(a.counters[0]) ^ 0xD80Full,
                                                     static_cast<uint64_t>(a.counters[1]),
                                                     static_cast<uint64_t>(a.counters[2]), a.dropout_salt)
                                           : 0ull;
    const uint32_t thr8 = dropout_thr8(a.dropout_p);
    const float keep_scale = dropout_scale8(thr8);
    const int n_pad = (a.N + 7) / 8 * 8;
    const int n_code = (a.N + 31) / 32 * 32;
    uint32_t pc = 0, asked = 0;  // panels done, residual panels asked for
    auto ask = [&](int64_t t, int p) {  // lane 0: the residual of panel p of tile t into buffer asked & 1
      const int b = asked & 1;
      mbar_expect_tx(&res_full[w][b], 4096);
      tma_load_2d(panel[b], &tmR, &res_full[w][b], static_cast<int>(t % n_tiles) * BN + col0 + p * 64,
                  static_cast<int>(t / n_tiles) * BM + quarter * 32);
    };
    if (a.residual) {
      if (lane == 0) ask(blockIdx.x, 0);
      asked = 1;
    }
    int lt = 0;
    bool stop = false;
    for (int64_t t = blockIdx.x; t < tiles && !stop; t += gridDim.x, ++lt) {
      const int m0 = static_cast<int>(t / n_tiles) * BM + quarter * 32, n0 = static_cast<int>(t % n_tiles) * BN;
      const int m = m0 + lane;
      const bool live = m < M;
      const bool slab_full = m0 + 32 <= M;  // rows past M are not written: no TMA store of such a slab
      const int ab = lt & 1;
      if (!mbar_wait(&acc_full[ab], (lt >> 1) & 1u, &abort_flag)) {
        if (lane == 0) set_error(a.err, kErrMmaTimeout);
        abort_flag = 1;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t trow = tmem_base + static_cast<uint32_t>(ab * BN) + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll 1
      for (int p = 0; p < S::kPanels; ++p, ++pc) {
        const int b = pc & 1;
        const int nc0 = n0 + col0 + p * 64;
        if (a.residual) {
          // the other buffer's store has been read: ask for the next panel into it
          const bool more = p + 1 < S::kPanels || t + gridDim.x < tiles;
          if (lane == 0) {
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            if (more) {
              if (p + 1 < S::kPanels)
                ask(t, p + 1);
              else
                ask(t + gridDim.x, 0);
            }
          }
          if (more) ++asked;
          if (!mbar_wait(&res_full[w][b], (pc >> 1) & 1u, &abort_flag)) {
            if (lane == 0) set_error(a.err, kErrMmaTimeout);
            abort_flag = 1;
            stop = true;
            break;
          }
        } else if (lane == 0) {
          // buffer b left two panels ago, the code panel one panel ago
          if (a.q8.q)
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          else
            asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
        }
        __syncwarp();
        if (nc0 < a.N) {
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            const int nc = nc0 + h * 32;
            float v[32];
            tmem_ld32(trow + static_cast<uint32_t>(col0 + p * 64 + h * 32), v);
            if (nc + 32 <= a.N) {
              if (a.bias) {
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] += __ldg(a.bias + nc + j);
              }
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = nc + j < a.N ? v[j] + (a.bias ? __ldg(a.bias + nc + j) : 0.f) : 0.f;
            }
            if (a.z && live) {
              __nv_bfloat16* dst = a.z + static_cast<int64_t>(m) * a.ldz + nc;
#pragma unroll
              for (int j = 0; j < 32; j += 8)
                if (nc + j < n_pad) *reinterpret_cast<uint4*>(dst + j) = f32_to_bf16x8(v + j);
            }
            if (a.q8.q && nc < n_code) {
              uint32_t mx = 0;
#pragma unroll
              for (int j = 0; j < 32; j += 8) mx = max(mx, abs_max_bits8(v + j));
              const uint32_t byte = group8_byte(mx);
              const float inv = group8_inv(byte);
              uint2 c[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) c[j] = a.act == kActRelu ? codes8_relu(v + 8 * j, inv) : codes8(v + 8 * j, inv);
              if (live) a.q8.e[static_cast<int64_t>(m) * a.q8.lde + (nc >> 5)] = static_cast<uint8_t>(byte);
              uint4* dst;
              if (slab_full) {
                // 64-byte rows in the 64B-swizzled layout of the store's map
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                  dst = reinterpret_cast<uint4*>(codes + lane * 64 + (((h * 2 + u) ^ ((lane >> 1) & 3)) << 4));
                  *dst = make_uint4(c[2 * u].x, c[2 * u].y, c[2 * u + 1].x, c[2 * u + 1].y);
                }
              } else if (live) {
                dst = reinterpret_cast<uint4*>(a.q8.q + static_cast<int64_t>(m) * a.q8.ldq + nc);
                dst[0] = make_uint4(c[0].x, c[0].y, c[1].x, c[1].y);
                dst[1] = make_uint4(c[2].x, c[2].y, c[3].x, c[3].y);
              }
            }
            if (a.act == kActRelu) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = v[j] < 0.f ? 0.f : v[j];  // a NaN stays
            } else if (a.act == kActGelu) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = gelu(v[j]);
            } else if (a.act == kActSilu) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = silu(v[j]);
            }
            if (a.dropout_p > 0.f) {
              const uint64_t base = static_cast<uint64_t>(m) * static_cast<uint64_t>(a.ldo) + static_cast<uint64_t>(nc);
              const uint32_t keep = dropout_keep_bits(key, base, 32, thr8);
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = (keep >> j) & 1u ? v[j] * keep_scale : 0.f;
            }
            uint8_t* prow = panel[b] + lane * 128;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint4* piece = reinterpret_cast<uint4*>(prow + (((h * 4 + q) ^ (lane & 7)) << 4));
              if (a.residual) {
                float r[8];
                bf16x8_to_f32(*piece, r);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[8 * q + j] = nc + 8 * q + j < a.N ? v[8 * q + j] + r[j] : 0.f;
              }
              if (slab_full)
                *piece = f32_to_bf16x8(v + 8 * q);
              else if (live && nc + 8 * q < n_pad)
                *reinterpret_cast<uint4*>(a.out + static_cast<int64_t>(m) * a.ldo + nc + 8 * q) = f32_to_bf16x8(v + 8 * q);
            }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          if (slab_full && nc0 < a.N) {
            tma_store_2d(&tmO, panel[b], nc0, m0);
            if (a.q8.q) tma_store_2d(&tmQ, codes, nc0, m0);
          }
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[ab]);
    }
    if (lane == 0) {
      // the panels are in shared memory that ends with the CTA: wait for the stores'
      // reads, and after an abort (bounded) for a residual panel still on its way
      asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      for (uint32_t i = pc; i < asked; ++i) {
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(&res_full[w][i & 1], (i >> 1) & 1u) && globaltimer_ns() - t0 < kWaitNs) {
        }
      }
    }
  }
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    tmem_dealloc(tmem_base, S::kTmemCols);
  }
}

template <int BN>
void launch_t(const LinearArgs& a, cudaStream_t stream) {
  using S = LSmem<BN>;
  const int64_t n_pad = ceil_div(a.N, 8) * 8;
  const CUtensorMap ma = tensor_map_bf16(a.A, a.a_rows, a.K, a.lda, BM);
  const CUtensorMap mw = tensor_map_bf16(a.W, a.N, a.K, a.ldw, BN);
  const CUtensorMap mo = tensor_map_bf16(a.out, a.out_rows, n_pad, a.ldo, 32);
  const CUtensorMap mr = a.residual ? tensor_map_bf16(a.residual, a.r_rows, n_pad, a.ldr, 32) : mo;
  const CUtensorMap mq =
      a.q8.q ? tensor_map_u8(a.q8.q, a.q_rows, ceil_div(a.N, 32) * 32, a.q8.ldq, 64, 32, CU_TENSOR_MAP_SWIZZLE_64B) : mo;
  auto kern = linear_fwd_kernel<BN>;
  set_smem(reinterpret_cast<const void*>(kern), S::kBytes);
  const int64_t tiles = ceil_div(a.cap, BM) * ceil_div(a.N, BN);
  launch_k(kern, dim3(static_cast<unsigned>(std::min<int64_t>(tiles, sm_count()))), dim3(S::kThreads), S::kBytes,
           stream, ma, mw, mr, mo, mq, a);
  GB_LAUNCH_CHECK();
}

}  // namespace

void launch_linear_fwd(const LinearArgs& a, cudaStream_t stream) {
  if (a.cap <= 0) return;
  // the widest tile that still gives every SM one: fewer re-reads of A, longer stores
  const int64_t mt = ceil_div(a.cap, BM);
  if (a.N > 128 && mt * ceil_div(a.N, 256) >= sm_count()) return launch_t<256>(a, stream);
  if (a.N > 64 && mt * ceil_div(a.N, 128) >= sm_count()) return launch_t<128>(a, stream);
  return launch_t<64>(a, stream);
}

}  // namespace dev
}  // namespace grappa
