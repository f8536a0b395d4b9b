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
//   warps 2..   epilogue: each warp owns 32 rows (a TMEM lane quarter) x 64 columns.  The
//               residual's panel comes by TMA into the very buffer that the output panel
//               leaves from (a lane adds and overwrites its own 16-byte pieces); the next
//               tile's is asked for as soon as that store has read the buffer.
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

// A warp of the epilogue owns 32 rows x 64 columns of the tile: one panel of output /
// residual.  The 256-wide tile takes a whole SM (16 epilogue warps);
// narrower tiles share it (2 and 3 CTAs), so that as many warps work on epilogues.
template <int BN>
struct LSmem {
  static constexpr int kEpi = BN / 16;                       // epilogue warps
  static constexpr int kCtas = BN == 256 ? 1 : (BN == 128 ? 2 : 3);
  static constexpr int kThreads = 64 + 32 * kEpi;
  static constexpr int kABytes = BM * BK * 2;
  static constexpr int kBBytes = BN * BK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kOutBytes = kEpi * 4096;              // a 32 x 64 bf16 panel a warp
  static constexpr int kBudget = 224 * 1024 / kCtas - 2048 - kOutBytes;
  static constexpr int kStages = kBudget / kStageBytes > 4 ? 4 : kBudget / kStageBytes;
  static constexpr int kTmemCols = 2 * BN;
  static constexpr int kBytes = kStages * kStageBytes + kOutBytes + 1024 /*align*/;
  static_assert(kStages >= 2 && kCtas * (kBytes + 1024) <= 227 * 1024 && kCtas * kTmemCols <= 512, "linear: resources");
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
__global__ void __launch_bounds__(LSmem<BN>::kThreads, LSmem<BN>::kCtas)
    linear_fwd_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                      const __grid_constant__ CUtensorMap tmR, const __grid_constant__ CUtensorMap tmO, LinearArgs a) {
  GB_PDL_ENTRY();
  using S = LSmem<BN>;
  constexpr int kStages = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full_bar[kStages], empty_bar[kStages], acc_full[2], acc_empty[2], res_full[S::kEpi];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;

  const int M = live_rows(a.n_ptr, a.cap);
  const int kbs = (a.K + BK - 1) / BK;
  const int n_tiles = (a.N + BN - 1) / BN;
  const int64_t tiles = static_cast<int64_t>((M + BM - 1) / BM) * n_tiles;
  if (static_cast<int64_t>(blockIdx.x) >= tiles) return;

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* out_area = smem + kStages * S::kStageBytes;
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
    }
    for (int w = 0; w < S::kEpi; ++w) mbar_init(&res_full[w], 1);
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
    const int col0 = (w / 4) * 64;
    uint8_t* panel = out_area + w * 4096;
    const uint64_t key = a.dropout_p > 0.f ? hop_key(static_cast<uint64_t>(a.counters[0]) ^ 0xD80Full,
                                                     static_cast<uint64_t>(a.counters[1]),
                                                     static_cast<uint64_t>(a.counters[2]), a.dropout_salt)
                                           : 0ull;
    const uint32_t thr8 = dropout_thr8(a.dropout_p);
    const float keep_scale = dropout_scale8(thr8);
    const bool bias16 = (reinterpret_cast<uintptr_t>(a.bias) & 15u) == 0;
    const int n_pad = (a.N + 7) / 8 * 8;
    const int n_code = (a.N + 31) / 32 * 32;
    auto ask = [&](int64_t t) {  // lane 0: tile t's residual panel
      mbar_expect_tx(&res_full[w], 4096);
      tma_load_2d(panel, &tmR, &res_full[w], static_cast<int>(t % n_tiles) * BN + col0,
                  static_cast<int>(t / n_tiles) * BM + quarter * 32);
    };
    if (a.residual && lane == 0) ask(blockIdx.x);
    int lt = 0, taken = 0;  // tiles begun, residual panels that have arrived
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x, ++lt) {
      const int m0 = static_cast<int>(t / n_tiles) * BM + quarter * 32, nc0 = static_cast<int>(t % n_tiles) * BN + col0;
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
      if (a.residual) {
        if (!mbar_wait(&res_full[w], lt & 1u, &abort_flag)) {
          if (lane == 0) set_error(a.err, kErrMmaTimeout);
          abort_flag = 1;
          break;
        }
        taken = lt + 1;
      } else {
        // the last tile's panels have left
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
      }
      const uint32_t trow =
          tmem_base + static_cast<uint32_t>(ab * BN + col0) + (static_cast<uint32_t>(quarter * 32) << 16);
      if (nc0 < a.N) {
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          const int nc = nc0 + h * 32;
          const bool whole = nc + 32 <= a.N;
          float v[32];
          tmem_ld32(trow + h * 32, v);
          if (whole) {
            if (a.bias) {
              if (bias16) {
#pragma unroll
                for (int j = 0; j < 32; j += 4) {
                  const float4 b4 = __ldg(reinterpret_cast<const float4*>(a.bias + nc + j));
                  v[j] += b4.x, v[j + 1] += b4.y, v[j + 2] += b4.z, v[j + 3] += b4.w;
                }
              } else {
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] += __ldg(a.bias + nc + j);
              }
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
            const float top = max_nan(abs_max3(abs_max8(v), abs_max8(v + 8), abs_max8(v + 16)), abs_max8(v + 24));
            const uint32_t byte = group8_byte(top);
            const float inv = group8_inv(byte);
            if (live) a.q8.e[static_cast<int64_t>(m) * a.q8.lde + (nc >> 5)] = static_cast<uint8_t>(byte);
            uint32_t c[8];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const uint2 cu = a.act == kActRelu ? codes8_relu(v + 8 * u, inv) : codes8(v + 8 * u, inv);
              c[2 * u] = cu.x, c[2 * u + 1] = cu.y;
            }
            // neighbouring lanes trade halves, so that a store writes whole 32-byte sectors:
            // first the even lane's row (16 bytes by each), then the odd lane's
            const bool odd = lane & 1;
            uint4 first, second;
            {
              uint32_t got[4];
#pragma unroll
              for (int u = 0; u < 4; ++u) got[u] = __shfl_xor_sync(0xffffffffu, odd ? c[u] : c[4 + u], 1);
              first = odd ? make_uint4(got[0], got[1], got[2], got[3]) : make_uint4(c[0], c[1], c[2], c[3]);
              second = odd ? make_uint4(c[4], c[5], c[6], c[7]) : make_uint4(got[0], got[1], got[2], got[3]);
            }
            const int me = m - (lane & 1);
            int8_t* dst = a.q8.q + static_cast<int64_t>(me) * a.q8.ldq + nc + (odd ? 16 : 0);
            if (me < M) *reinterpret_cast<uint4*>(dst) = first;
            if (me + 1 < M) *reinterpret_cast<uint4*>(dst + a.q8.ldq) = second;
          }
          if (a.act == kActRelu) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = v[j] < 0.f ? 0.f : v[j];  // a NaN stays
          } else if (a.act == kActGelu) {
#pragma unroll
            for (int j = 0; j < 32; j += 2) gelu2(v + j);
          } else if (a.act == kActSilu) {
#pragma unroll
            for (int j = 0; j < 32; j += 2) silu2(v + j);
          }
          if (a.dropout_p > 0.f) {
            const uint64_t base = static_cast<uint64_t>(m) * static_cast<uint64_t>(a.ldo) + static_cast<uint64_t>(nc);
            const uint32_t keep = dropout_keep_bits(key, base, 32, thr8);
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = (keep >> j) & 1u ? v[j] * keep_scale : 0.f;
          }
          uint8_t* prow = panel + lane * 128;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint4* piece = reinterpret_cast<uint4*>(prow + (((h * 4 + q) ^ (lane & 7)) << 4));
            if (a.residual) {
              float r[8];
              bf16x8_to_f32(*piece, r);
#pragma unroll
              for (int j = 0; j < 8; ++j) v[8 * q + j] += r[j];
              if (!whole) mask8(v + 8 * q, (nc >> 3) + q, a.N);
            }
            if (slab_full)
              *piece = f32_to_bf16x8(v + 8 * q);
            else if (live && nc + 8 * q < n_pad)
              *reinterpret_cast<uint4*>(a.out + static_cast<int64_t>(m) * a.ldo + nc + 8 * q) = f32_to_bf16x8(v + 8 * q);
          }
        }
      }
      // the accumulator is read: the products of the tile after the next may start
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&acc_empty[ab]);
        if (slab_full && nc0 < a.N) tma_store_2d(&tmO, panel, nc0, m0);
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        if (a.residual && t + gridDim.x < tiles) {
          asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          ask(t + gridDim.x);
        }
      }
    }
    if (lane == 0) {
      // the panels are in shared memory that ends with the CTA: wait for the stores'
      // reads, and after an abort (bounded) for a residual panel still on its way
      asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      if (abort_flag && a.residual) {
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(&res_full[w], taken & 1u) && globaltimer_ns() - t0 < kWaitNs) {
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
  auto kern = linear_fwd_kernel<BN>;
  set_smem(reinterpret_cast<const void*>(kern), S::kBytes);
  const int64_t tiles = ceil_div(a.cap, BM) * ceil_div(a.N, BN);
  launch_k(kern, dim3(static_cast<unsigned>(std::min<int64_t>(tiles, sm_count() * S::kCtas))), dim3(S::kThreads), S::kBytes,
           stream, ma, mw, mr, mo, a);
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
