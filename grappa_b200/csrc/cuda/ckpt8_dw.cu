// Weight gradient from rows kept in 8 bits: gW[M][N] (+)= dY^T Xh, Xh the rows that the
// codes stand for, exact in bf16.  The reduction runs over the rows, so both operands are
// MN-major and read in place.
//
// A CTA computes a (128 MT) x NT tile over a share of the rows, 32 at a time:
//   warp 0      TMA producer: dY boxes straight into the MMA's layout, codes (128-byte
//               rows, swizzled) beside them
//   warps 2..17 turn the codes into the bf16 operand, four teams of four in turn: a warp
//               takes groups of 32 columns, a lane one row (32 bytes of codes, one
//               exponent byte), and writes 64 bytes in the 128B-swizzled layout; later the
//               epilogue
//   warp 1      issues tcgen05.mma into MT accumulators of NT TMEM columns
// The bf16 form of the rows never leaves the SM: HBM sees dY once and a byte a value.
//
// Accuracy: the tensor core adds into its fp32 accumulator by truncation, so a sum over R
// rows drifts by about 1.2e-9 R of itself (measured on the bf16 GEMM: 1.6e-4 at 139058 rows,
// 4e-6 at 3758).  The accumulator is therefore emptied every kChainRows rows into the CTA's own partial
// tile, in fp32 with rounding to nearest (the first time a store, then reductions that
// this thread alone makes to these addresses, so their order is fixed).  A second kernel
// adds the CTAs' partial tiles in order: the same bits every time.
#include <algorithm>

#include "ckpt8.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace grappa {
namespace dev {

namespace {

constexpr int BK = 32;            // rows of a block
constexpr int kConv = 16;         // converter / epilogue warps, in four teams of
constexpr int kTeam = 4;
constexpr int kTeams = kConv / kTeam;
constexpr int kThreads = 64 + 32 * kConv;
constexpr int kAhead = 2;
constexpr int kChainRows = 4096;
constexpr int kChainKb = kChainRows / BK;

template <int MT, int NT>
struct DSmem {
  static constexpr int kABytes = MT * 128 * BK * 2;
  static constexpr int kRawBytes = NT * BK;
  static constexpr int kBBytes = NT * BK * 2;
  static constexpr int kSlotBytes = kABytes + kRawBytes;
  static constexpr int kBSlots = kTeams;
  static constexpr int kBudget = 224 * 1024 - kBSlots * kBBytes;
  static constexpr int kSlots = kBudget / kSlotBytes > 12 ? 12 : kBudget / kSlotBytes;
  static constexpr int kTmemCols = MT * NT;
  static constexpr int kBytes = kSlots * kSlotBytes + kBSlots * kBBytes + 1024 /*align*/;
  static_assert(kSlots >= 3 && kTmemCols <= 512 && kBytes <= 226 * 1024, "ckpt8_dw: shared memory");
};

// How the rows are shared: kb_total blocks of BK rows over `splits` CTAs a tile, fewer
// when the live rows are few (each then takes at least min_kb blocks).
struct Shares {
  int splits, per;
};
__host__ __device__ inline Shares shares(int kb_total, int splits_max, int min_kb) {
  int s = kb_total / min_kb;
  s = s < 1 ? 1 : (s > splits_max ? splits_max : s);
  const int per = (kb_total + s - 1) / s;
  s = per > 0 ? (kb_total + per - 1) / per : 1;
  return {s < 1 ? 1 : s, per};
}

struct DwPlan {
  int mt, nt;            // tile: 128 mt x nt
  int m_tiles, n_tiles;
  int splits, min_kb;
  bool y_blocks = false, q_blocks = false;  // operands of whole column blocks (64 bf16, 128 codes)
};

template <int MT, int NT>
__global__ void __launch_bounds__(kThreads, 1)
    ckpt8_dw_kernel(const __grid_constant__ CUtensorMap tmY, const __grid_constant__ CUtensorMap tmQ, Ckpt8DwArgs a,
                    DwPlan plan) {
  GB_PDL_ENTRY();
  using S = DSmem<MT, NT>;
  constexpr int kSlots = S::kSlots;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full_bar[kSlots], empty_bar[kSlots], b_full[kTeams], b_empty[kTeams], acc_full, acc_empty;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;

  const int n = live_rows(a.n_ptr, a.cap);
  const int kb_total = (n + BK - 1) / BK;
  const Shares sh = shares(kb_total, plan.splits, plan.min_kb);
  const int tile = blockIdx.x % (plan.m_tiles * plan.n_tiles), split = blockIdx.x / (plan.m_tiles * plan.n_tiles);
  if (split >= sh.splits) return;
  const int m0 = (tile / plan.n_tiles) * (128 * MT), n0 = (tile % plan.n_tiles) * NT;
  const int kb0 = split * sh.per, kb1 = min(kb_total, kb0 + sh.per);
  float* part = a.work + static_cast<int64_t>(blockIdx.x) * (128 * MT * NT);

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* b_area = smem + kSlots * S::kSlotBytes;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < kTeams; ++b) {
      mbar_init(&b_full[b], kTeam);
      mbar_init(&b_empty[b], 1);
    }
    mbar_init(&acc_full, 1);
    mbar_init(&acc_empty, kConv);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(&tmem_slot, S::kTmemCols);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = tmem_slot;
  const int nkb = max(0, kb1 - kb0);

  if (warp == 0) {
    if (lane == 0) {
      int issued = 0;
      for (int i = 0; i < nkb; ++i) {
        const int s = i % kSlots;
        if (i >= kSlots && !mbar_wait(&empty_bar[s], ((i / kSlots) & 1u) ^ 1u, &abort_flag)) {
          set_error(a.err, kErrMmaTimeout);
          abort_flag = 1;
          break;
        }
        uint8_t* sa = smem + s * S::kSlotBytes;
        uint8_t* sq = sa + S::kABytes;
        const int r0 = (kb0 + i) * BK;
        mbar_expect_tx(&full_bar[s], S::kSlotBytes);
        // whole column blocks: one load an operand
        if (plan.y_blocks) {
          tma_load_3d(sa, &tmY, &full_bar[s], 0, r0, m0 / 64);
        } else {
#pragma unroll
          for (int c = 0; c < 2 * MT; ++c) tma_load_2d(sa + c * (64 * BK * 2), &tmY, &full_bar[s], m0 + c * 64, r0);
        }
        if (plan.q_blocks) {
          tma_load_3d(sq, &tmQ, &full_bar[s], 0, r0, n0 / 128);
        } else {
#pragma unroll
          for (int c = 0; c < NT / 128; ++c) tma_load_2d(sq + c * (128 * BK), &tmQ, &full_bar[s], n0 + c * 128, r0);
        }
        issued = i + 1;
      }
      if (abort_flag) {
        for (int i = issued > kSlots ? issued - kSlots : 0; i < issued; ++i) {
          const uint64_t t0 = globaltimer_ns();
          while (!mbar_try_wait(&full_bar[i % kSlots], (i / kSlots) & 1u) && globaltimer_ns() - t0 < kWaitNs) {
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = umma_idesc(128, NT, true, true);
      int chunk = 0;
      for (int i = 0; i < nkb; ++i) {
        const int s = i % kSlots, b = i % kTeams;
        const bool first = i % kChainKb == 0;
        // the accumulator of the last chain has been read
        if (first && chunk > 0 && !mbar_wait(&acc_empty, (chunk - 1) & 1u, &abort_flag)) {
          set_error(a.err, kErrMmaTimeout);
          abort_flag = 1;
          break;
        }
        // dY's tile (the loads' own barrier) and the converted rows
        if (!mbar_wait(&full_bar[s], (i / kSlots) & 1u, &abort_flag) ||
            !mbar_wait(&b_full[b], (i / kTeams) & 1u, &abort_flag)) {
          set_error(a.err, kErrMmaTimeout);
          abort_flag = 1;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t sa = smem_u32(smem + s * S::kSlotBytes), sb = smem_u32(b_area + b * S::kBBytes);
#pragma unroll
        for (int kk = 0; kk < BK / 16; ++kk) {
          const uint64_t db = umma_desc(sb + kk * 2048, 64 * BK * 2, 1024);
#pragma unroll
          for (int h = 0; h < MT; ++h)
            umma_f16(tmem_base + h * NT, umma_desc(sa + h * (128 * BK * 2) + kk * 2048, 64 * BK * 2, 1024), db, idesc,
                     (!first || kk > 0) ? 1u : 0u);
        }
        umma_commit(&empty_bar[s]);
        umma_commit(&b_empty[b]);
        if (i % kChainKb == kChainKb - 1 || i == nkb - 1) {
          umma_commit(&acc_full);
          ++chunk;
        }
      }
    }
  } else {
    // the teams take the blocks in turn, each with an operand slot of its own: a team has four
    // MMA times for a block, and one's waits overlap the others' arithmetic
    const int w = warp - 2;
    constexpr int kGroups = NT / 32;
    constexpr int kItems = kGroups / kTeam;  // groups of a warp
    const int b = w / kTeam, w4 = w % kTeam;
    uint8_t* sb = b_area + b * S::kBBytes;
    // exponent bytes come from global memory: asked for kAhead own blocks ahead
    uint32_t byte[kAhead][kItems];
    auto fetch = [&](int i, uint32_t (&to)[kItems]) {
#pragma unroll
      for (int u = 0; u < kItems; ++u) {
        const int g = n0 / 32 + w4 + u * kTeam, r = (kb0 + i) * BK + lane;
        to[u] = (i < nkb && r < n && g < a.groups) ? __ldg(a.q8.e + static_cast<int64_t>(r) * a.q8.lde + g) : 0u;
      }
    };
#pragma unroll
    for (int p = 0; p < kAhead; ++p) fetch(b + kTeams * p, byte[p]);
    int i = b;
    bool stop = false;
    for (int chunk = 0; chunk * kChainKb < nkb && !stop; ++chunk) {
      const int end = min(nkb, (chunk + 1) * kChainKb);
      for (; i < end; i += kTeams) {
        const int s = i % kSlots;
        const int r0 = (kb0 + i) * BK;
        bool ok = mbar_wait(&full_bar[s], (i / kSlots) & 1u, &abort_flag);
        if (ok && i >= kTeams) ok = mbar_wait(&b_empty[b], (i / kTeams - 1) & 1u, &abort_flag);
        if (!ok) {
          if (lane == 0) set_error(a.err, kErrMmaTimeout);
          abort_flag = 1;
          stop = true;
          break;
        }
        uint8_t* sa = smem + s * S::kSlotBytes;
        const uint8_t* sq = sa + S::kABytes;
#pragma unroll
        for (int u = 0; u < kItems; ++u) {
          const int g = w4 + u * kTeam, k = lane;
          const __nv_bfloat162 scale = group8_scale_bf16(byte[0][u]);
          // codes: box g / 4 of 128-byte rows, 16-byte pieces 2 (g % 4) + 0, 1, swizzled
          const uint8_t* row = sq + (g >> 2) * (128 * BK) + k * 128;
          // operand: box g / 2 of 64 columns, pieces 4 (g % 2) + 0..3, swizzled
          uint8_t* out = sb + (g >> 1) * (64 * BK * 2) + k * 128;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint4 c = *reinterpret_cast<const uint4*>(row + ((((g & 3) * 2 + h) ^ (k & 7)) << 4));
            uint4 v0 = values8_bf16(c.x, c.y, scale), v1 = values8_bf16(c.z, c.w, scale);
            if (r0 + k >= n) v0 = v1 = make_uint4(0u, 0u, 0u, 0u);
            *reinterpret_cast<uint4*>(out + ((((g & 1) * 4 + h * 2) ^ (k & 7)) << 4)) = v0;
            *reinterpret_cast<uint4*>(out + ((((g & 1) * 4 + h * 2 + 1) ^ (k & 7)) << 4)) = v1;
          }
        }
#pragma unroll
        for (int p = 0; p + 1 < kAhead; ++p)
#pragma unroll
          for (int u = 0; u < kItems; ++u) byte[p][u] = byte[p + 1][u];
        fetch(i + kTeams * kAhead, byte[kAhead - 1]);
        // rows past the live ones may hold anything: their dY is zeroed here
        if (r0 + BK > n) {
          for (int x = w4 * 32 + lane; x < 2 * MT * BK; x += kTeam * 32) {
            const int k = x % BK;
            if (r0 + k >= n) {
              uint4* p = reinterpret_cast<uint4*>(sa + (x / BK) * (64 * BK * 2) + k * 128);
#pragma unroll
              for (int q = 0; q < 8; ++q) p[q] = make_uint4(0u, 0u, 0u, 0u);
            }
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&b_full[b]);
      }
      if (stop) break;
      if (!mbar_wait(&acc_full, chunk & 1u, &abort_flag)) {
        if (lane == 0) set_error(a.err, kErrMmaTimeout);
        abort_flag = 1;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      // warp w: TMEM lanes of its quarter, a fourth of the MT * NT columns.  The partial tile
      // is laid out as the warp writes it: 32 columns at a time, 4 of them a lane and
      // store, 512 bytes a store
      const int quarter = warp & 3, share = w >> 2;
#pragma unroll 1
      for (int c = share * (MT * NT / 4); c < (share + 1) * (MT * NT / 4); c += 32) {
        float v[32];
        tmem_ld32(tmem_base + static_cast<uint32_t>(c) + (static_cast<uint32_t>(quarter * 32) << 16), v);
        float* p = part + (static_cast<int64_t>(c / 32) * 4 + quarter) * 1024 + lane * 4;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (chunk == 0)
            *reinterpret_cast<float4*>(p + j * 128) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          else
            red_add_v4(p + j * 128, v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty);
    }
  }
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    tmem_dealloc(tmem_base, S::kTmemCols);
  }
}

// gW (+)= the partial tiles of the splits, in order.  One thread per four columns of a row
// of a tile, in the partial tiles' own order.
__global__ void __launch_bounds__(256) ckpt8_dw_sum_kernel(Ckpt8DwArgs a, DwPlan plan) {
  GB_PDL_ENTRY();
  const int n = live_rows(a.n_ptr, a.cap);
  const int kb_total = (n + BK - 1) / BK;
  const int splits = kb_total > 0 ? shares(kb_total, plan.splits, plan.min_kb).splits : 0;
  const int tile_floats = 128 * plan.mt * plan.nt;
  const int tiles = plan.m_tiles * plan.n_tiles;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int tile = static_cast<int>(i / (tile_floats / 4));
  if (tile >= tiles) return;
  const int at = static_cast<int>(i % (tile_floats / 4)) * 4;
  // at = ((c / 32) * 4 + quarter) * 1024 + j * 128 + lane * 4
  const int lane = (at / 4) % 32, j = (at / 128) % 8, quarter = (at / 1024) % 4, c32 = at / 4096;
  const int col_t = c32 * 32 + j * 4;  // column over the MT accumulators
  const int m = (tile / plan.n_tiles) * 128 * plan.mt + (col_t / plan.nt) * 128 + quarter * 32 + lane;
  const int nn = (tile % plan.n_tiles) * plan.nt + col_t % plan.nt;
  if (m >= a.M || nn >= a.N) return;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  const float* p = a.work + static_cast<int64_t>(tile) * tile_floats + at;
#pragma unroll 8
  for (int k = 0; k < splits; ++k) {
    const float4 v = *reinterpret_cast<const float4*>(p + static_cast<int64_t>(k) * tiles * tile_floats);
    s.x += v.x;
    s.y += v.y;
    s.z += v.z;
    s.w += v.w;
  }
  float* g = a.gw + static_cast<int64_t>(m) * a.ldg + nn;
  const float o[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (nn + q < a.N) g[q] = (a.accumulate ? g[q] : 0.f) + o[q];
}

// Tile and shares for M x N over cap rows on num_sms SMs.  The large tile (256 x 256) reads
// each operand least often and converts each code once per 256 columns of dY; it needs
// enough rows for every SM to get some 32 blocks of them.  With fewer rows the small tile
// spreads the same work over four times as many CTAs.
DwPlan plan_for(int M, int N, int cap, int num_sms) {
  DwPlan p;
  const int64_t kb = ceil_div(std::max(cap, 1), BK);
  p.mt = M > 128 ? 2 : 1;
  p.nt = N > 128 ? 256 : 128;
  p.min_kb = 16;
  if (ceil_div(M, 128 * p.mt) * ceil_div(N, p.nt) * kb < 32ll * num_sms) {
    p.mt = 1;
    p.nt = 128;
    p.min_kb = 8;
  }
  p.m_tiles = static_cast<int>(ceil_div(M, 128 * p.mt));
  p.n_tiles = static_cast<int>(ceil_div(N, p.nt));
  const int64_t tiles = static_cast<int64_t>(p.m_tiles) * p.n_tiles;
  p.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(num_sms / tiles, kb / p.min_kb)));
  return p;
}

template <int MT, int NT>
void launch_t(const Ckpt8DwArgs& a, DwPlan p, cudaStream_t stream) {
  using S = DSmem<MT, NT>;
  p.y_blocks = a.dy_cols % 64 == 0;
  p.q_blocks = a.q_cols % 128 == 0;
  const CUtensorMap my = p.y_blocks ? tensor_map_blocks(CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.dy, a.dy_rows, a.dy_cols,
                                                        a.lddy, 64, BK, 2 * MT)
                                    : tensor_map_bf16(a.dy, a.dy_rows, a.dy_cols, a.lddy, BK);
  const CUtensorMap mq =
      p.q_blocks ? tensor_map_blocks(CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.q8.q, a.q_rows, a.q_cols, a.q8.ldq, 128, BK, NT / 128)
                 : tensor_map_u8(a.q8.q, a.q_rows, a.q_cols, a.q8.ldq, 128, BK, CU_TENSOR_MAP_SWIZZLE_128B);
  auto kern = ckpt8_dw_kernel<MT, NT>;
  set_smem(reinterpret_cast<const void*>(kern), S::kBytes);
  launch_k(kern, dim3(static_cast<unsigned>(p.m_tiles * p.n_tiles * p.splits)), dim3(kThreads), S::kBytes, stream, my,
           mq, a, p);
  GB_LAUNCH_CHECK();
}

}  // namespace

int64_t ckpt8_dw_work_floats(int M, int N, int cap, int num_sms) {
  const DwPlan p = plan_for(M, N, cap, num_sms);
  return static_cast<int64_t>(p.m_tiles) * p.n_tiles * p.splits * 128 * p.mt * p.nt;
}

void launch_ckpt8_dw(const Ckpt8DwArgs& a, int num_sms, cudaStream_t stream) {
  const DwPlan p = plan_for(a.M, a.N, a.cap, num_sms);
  if (p.mt == 2)
    p.nt == 256 ? launch_t<2, 256>(a, p, stream) : launch_t<2, 128>(a, p, stream);
  else
    p.nt == 256 ? launch_t<1, 256>(a, p, stream) : launch_t<1, 128>(a, p, stream);
  const int64_t threads = static_cast<int64_t>(p.m_tiles) * p.n_tiles * 128 * p.mt * p.nt / 4;
  launch_k(ckpt8_dw_sum_kernel, dim3(static_cast<unsigned>(ceil_div(threads, 256))), dim3(256), 0, stream, a, p);
  GB_LAUNCH_CHECK();
}

}  // namespace dev
}  // namespace grappa
