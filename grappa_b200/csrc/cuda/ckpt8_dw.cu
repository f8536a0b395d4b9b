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
constexpr int kClusterKb = 48;     // blocks a split at most where the splits are a cluster
static_assert(kClusterKb * BK <= 2048, "one chain");
constexpr int kChainRows = 2048;
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
  static_assert(kSlots >= kTeams && kTmemCols <= 512 && kBytes <= 226 * 1024, "ckpt8_dw: shared memory");
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
  int rows;              // of a block
  int splits, min_kb;    // CTAs (pairs) a tile at most, blocks each at least
  bool pair = false;     // by CTA pairs (mt = 2, nt = 256)
  bool cluster = false;  // a tile's splits are one cluster that sums its partial tiles itself
  bool y_blocks = false, q_blocks = false;  // operands of whole column blocks (64 bf16, 128 codes)
};

// Four sums into row m, columns nn .. nn + 3 of gW.
__device__ __forceinline__ void add_quad(const Ckpt8DwArgs& a, int m, int nn, float4 s) {
  if (m >= a.M || nn >= a.N) return;
  float* g = a.gw + static_cast<int64_t>(m) * a.ldg + nn;
  if (nn + 4 <= a.N && (reinterpret_cast<uintptr_t>(g) & 15) == 0) {
    float4* g4 = reinterpret_cast<float4*>(g);
    if (a.accumulate) {
      const float4 o = *g4;
      s.x += o.x, s.y += o.y, s.z += o.z, s.w += o.w;
    }
    *g4 = s;
    return;
  }
  const float o[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (nn + q < a.N) g[q] = (a.accumulate ? g[q] : 0.f) + o[q];
}

template <int MT, int NT>
__global__ void __launch_bounds__(kThreads, 1)
    ckpt8_dw_kernel(const __grid_constant__ CUtensorMap tmY, const __grid_constant__ CUtensorMap tmQ, Ckpt8DwArgs a,
                    DwPlan plan) {
  using S = DSmem<MT, NT>;
  constexpr int kSlots = S::kSlots;
  const bool cluster = MT == 1 && NT == 128 && plan.cluster;  // only the small tile's plans set it
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full_bar[kSlots], empty_bar[kSlots], b_full[kTeams], b_empty[kTeams], acc_full, acc_empty;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;

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
    prefetch_map(&tmY);
    prefetch_map(&tmQ);
  }
  if (warp == 1) tmem_alloc(&tmem_slot, S::kTmemCols);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = tmem_slot;
  // all of this may run while the kernel before is ending; its results are read from here on
  GB_PDL_ENTRY();
  const int n = live_rows(a.n_ptr, a.cap);
  const int kb_total = (n + BK - 1) / BK;
  const Shares sh = shares(kb_total, plan.splits, plan.min_kb);
  // the splits of a tile are a cluster (plan.cluster), or tiles apart
  const int tiles = plan.m_tiles * plan.n_tiles;
  const int tile = cluster ? blockIdx.x / plan.splits : blockIdx.x % tiles;
  const int split = cluster ? blockIdx.x % plan.splits : blockIdx.x / tiles;
  const int m0 = (tile / plan.n_tiles) * (128 * MT), n0 = (tile % plan.n_tiles) * NT;
  const int kb0 = split * sh.per, kb1 = split < sh.splits ? min(kb_total, kb0 + sh.per) : kb0;
  float* part = a.work + static_cast<int64_t>(blockIdx.x) * (128 * MT * NT);
  const int nkb = max(0, kb1 - kb0);

  // the two issuing warps stay converged; one elected lane issues (elect_one)
  if (warp == 0) {
    int issued = 0;
    for (int i = 0; i < nkb; ++i) {
      const int s = i % kSlots;
      if (i >= kSlots && !mbar_wait_all(&empty_bar[s], ((i / kSlots) & 1u) ^ 1u, &abort_flag)) {
        if (lane == 0) set_error(a.err, kErrMmaTimeout);
        abort_flag = 1;
        break;
      }
      uint8_t* sa = smem + s * S::kSlotBytes;
      uint8_t* sq = sa + S::kABytes;
      const int r0 = (kb0 + i) * BK;
      if (elect_one()) {
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
      }
      __syncwarp();
      issued = i + 1;
    }
    if (abort_flag) {
      for (int i = issued > kSlots ? issued - kSlots : 0; i < issued; ++i) {
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(&full_bar[i % kSlots], (i / kSlots) & 1u) && globaltimer_ns() - t0 < kWaitNs) {
        }
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = umma_idesc(128, NT, true, true);
    int chunk = 0;
    for (int i = 0; i < nkb; ++i) {
      const int s = i % kSlots, b = i % kTeams;
      const bool first = i % kChainKb == 0;
      // the accumulator of the last chain has been read; dY's tile (the loads' own barrier)
      // and the converted rows have come
      if ((first && chunk > 0 && !mbar_wait_all(&acc_empty, (chunk - 1) & 1u, &abort_flag)) ||
          !mbar_wait_all(&full_bar[s], (i / kSlots) & 1u, &abort_flag) ||
          !mbar_wait_all(&b_full[b], (i / kTeams) & 1u, &abort_flag)) {
        if (lane == 0) set_error(a.err, kErrMmaTimeout);
        abort_flag = 1;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t sa = smem_u32(smem + s * S::kSlotBytes), sb = smem_u32(b_area + b * S::kBBytes);
      const bool last = i % kChainKb == kChainKb - 1 || i == nkb - 1;
      if (elect_one()) {
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
        if (last) umma_commit(&acc_full);
      }
      __syncwarp();
      if (last) ++chunk;
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
        // the operand slot first: its last block's products are done, so block i - kSlots has
        // come (a wait by parity must not begin two phases early, and loads may complete out
        // of order)
        bool ok = i < kTeams || mbar_wait_all(&b_empty[b], (i / kTeams - 1) & 1u, &abort_flag);
        ok = ok && mbar_wait_all(&full_bar[s], (i / kSlots) & 1u, &abort_flag);
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
      if (!mbar_wait_all(&acc_full, chunk & 1u, &abort_flag)) {
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
        if (cluster) {
          // a cluster's CTA keeps it in its own shared memory, where the ring was (its only
          // chain is over, so every load and product of the ring is), row by row, pieces of 4
          // columns swizzled
          float4* t = reinterpret_cast<float4*>(smem) + (quarter * 32 + lane) * 32;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            t[(c / 4 + j) ^ lane] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          continue;
        }
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
  if (cluster) {
    // gW (+)= the cluster's partial tiles, in order, each CTA a share of the tile
    cluster_sync();
    // (a warp 128 columns of a row: whole lines of gW)
    constexpr int kQuads = 128 * 128 / 4;
    const int splits = kb_total > 0 ? sh.splits : 0;
    for (int x = split * kThreads + static_cast<int>(threadIdx.x); x < kQuads; x += plan.splits * kThreads) {
      const int row = x / 32, k = x % 32;
      const uint8_t* at = smem + (row * 32 + (k ^ (row & 31))) * 16;
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
      float4 v[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        v[r] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < splits) v[r] = ld_cluster4(cluster_addr(at, static_cast<uint32_t>(r)));
      }
#pragma unroll
      for (int r = 0; r < 8; ++r) s.x += v[r].x, s.y += v[r].y, s.z += v[r].z, s.w += v[r].w;
      add_quad(a, m0 + row, n0 + k * 4, s);
    }
    cluster_sync();  // the others may still read this CTA's tile
  }
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    tmem_dealloc(tmem_base, S::kTmemCols);
  }
}

// ---------------------------------------------------------------- CTA pairs
// The large tile (256 x 256) by two CTAs (cta_group::2): each loads 128 columns of dY and
// 128 columns of codes, converts its own, and the products read both CTAs' operands.  Per
// SM that halves the operand bytes that the tensor core reads from shared memory (which
// bound the single CTA: 96 KB of traffic a 32-row block against 512 cycles of products),
// and the accumulator takes half of TMEM, so there are two: four warps of their own empty
// one while the products of the next 2048 rows fill the other.
//   warp 0        TMA producer of dY: 128 columns a CTA, on CTA 0's barrier
//   warp 1        (CTA 0) issues the products
//   warp 2        TMA producer of the codes, on the CTA's own barriers
//   warps 3..18   converters, four warps a block (32 rows x 64 columns each), one team of
//                 them for every operand slot
//   warps 19..22  epilogue
// dY, codes and converted rows have rings of their own, each as long as its way round wants:
// dY is held from its load (some 2800 cycles under load) to the end of its products, the
// codes until they are converted, the operand from there to the end of the products.  One
// commit a block, to both CTAs, says that its products are done.  (With one ring of 5 slots
// for all three the way round was 4100 cycles without any work, 820 a block; two commits a
// 32-row block kept the issuing thread busy for 1900 cycles.)  The last block of a partly
// filled 64 rows takes its dY through the converters, which write zeros for the rows past
// the live ones.
struct PairSmem {
  static constexpr int kRows = 64;
  static constexpr int kYBytes = 128 * kRows * 2, kYSlots = 7;
  static constexpr int kBBytes = 128 * kRows * 2, kBSlots = 4;
  static constexpr int kQBytes = 128 * kRows, kQSlots = 5;
  static constexpr int kDone = 8;                            // barriers of finished blocks
  static constexpr int kTeamW = 4;                           // warps of a team
  static constexpr int kWarps = 3 + kBSlots * kTeamW + 4;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kChain = kChainRows / kRows;
  static constexpr int kBytes = kYSlots * kYBytes + kBSlots * kBBytes + kQSlots * kQBytes + 1024 /*align*/;
  static_assert(kBytes <= 226 * 1024 && kDone >= kYSlots && kQSlots > kBSlots, "ckpt8_dw pair: shared memory");
};

__global__ void __launch_bounds__(PairSmem::kThreads, 1)
    ckpt8_dw_pair_kernel(const __grid_constant__ CUtensorMap tmY, const __grid_constant__ CUtensorMap tmQ,
                         Ckpt8DwArgs a, DwPlan plan) {
  using S = PairSmem;
  constexpr int kYSlots = S::kYSlots, kBSlots = S::kBSlots, kQSlots = S::kQSlots, kDone = S::kDone;
  constexpr int kRows = S::kRows, kChain = S::kChain;
  constexpr int NT = 256;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t y_full[kYSlots], b_full[kBSlots], q_full[kQSlots], q_empty[kQSlots], done_bar[kDone], acc_full[2],
      acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* b_area = smem + kYSlots * S::kYBytes;
  uint8_t* q_area = b_area + kBSlots * S::kBBytes;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kYSlots; ++s) mbar_init(&y_full[s], 1);
    for (int s = 0; s < kBSlots; ++s) mbar_init(&b_full[s], 2 * S::kTeamW);  // the block's team in either CTA
    for (int s = 0; s < kQSlots; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], S::kTeamW);
    }
    for (int s = 0; s < kDone; ++s) mbar_init(&done_bar[s], 1);
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 8);  // four warps in either CTA
    }
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_map(&tmY);
    prefetch_map(&tmQ);
  }
  if (warp == 1) tmem_alloc_pair(&tmem_slot, 2 * NT);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = tmem_slot;

  // all of this may run while the kernel before is ending; its results are read from here on
  GB_PDL_ENTRY();
  const int n = live_rows(a.n_ptr, a.cap);
  const int kb_total = (n + kRows - 1) / kRows;
  const Shares sh = shares(kb_total, plan.splits, plan.min_kb);
  const int pair = blockIdx.x >> 1, rank = static_cast<int>(cluster_rank());
  const int tile = pair % (plan.m_tiles * plan.n_tiles), split = pair / (plan.m_tiles * plan.n_tiles);
  const int m0 = (tile / plan.n_tiles) * 256 + rank * 128, n0 = (tile % plan.n_tiles) * NT + rank * 128;
  // the splits take the blocks in turn, so that the whole device reads one stretch of rows
  const int nkb = split < sh.splits && kb_total > split ? (kb_total - split + sh.splits - 1) / sh.splits : 0;
  auto row0 = [&](int i) { return (split + i * sh.splits) * kRows; };
  // number of the partly filled block (-1: none here)
  const int tail = n % kRows != 0 && nkb > 0 && row0(nkb - 1) + kRows > n ? nkb - 1 : -1;
  float* part = a.work + static_cast<int64_t>(blockIdx.x) * (128 * NT);
  // waits until the products of the pair's block j are done (j in order for every caller,
  // or after a later block: a wait by parity must not begin two phases early)
  auto products_done = [&](int j) { return mbar_wait_all(&done_bar[j % kDone], (j / kDone) & 1u, &abort_flag); };
  // the three issuing warps stay converged; one elected lane issues (elect_one)
  if (warp == 0) {
    int issued = 0;
    for (int i = 0; i < nkb; ++i) {
      const int s = i % kYSlots;
      if (i >= kYSlots && !products_done(i - kYSlots)) {
        if (lane == 0) set_error(a.err, kErrMmaTimeout);
        abort_flag = 1;
        break;
      }
      uint8_t* sy = smem + s * S::kYBytes;
      const int r0 = row0(i);
      if (elect_one()) {
        if (i == tail) {
          if (rank == 0) mbar_arrive(&y_full[s]);
        } else {
          if (rank == 0) mbar_expect_tx(&y_full[s], 2 * S::kYBytes);
          const uint32_t bar = cluster_addr(&y_full[s], 0);
          tma_load_2d_pair(sy, &tmY, bar, m0, r0);
          tma_load_2d_pair(sy + 64 * kRows * 2, &tmY, bar, m0 + 64, r0);
        }
      }
      __syncwarp();
      if (i != tail) issued = i + 1;
    }
    if (abort_flag && rank == 0) {
      for (int i = issued > kYSlots ? issued - kYSlots : 0; i < issued; ++i) {
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(&y_full[i % kYSlots], (i / kYSlots) & 1u) && globaltimer_ns() - t0 < kWaitNs) {
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      constexpr uint32_t idesc = umma_idesc(256, NT, true, true);
      for (int i = 0; i < nkb; ++i) {
        const int s = i % kYSlots, b = i % kBSlots;
        const int chain = i / kChain, ab = chain & 1;
        const bool first = i % kChain == 0;
        if ((first && chain >= 2 && !mbar_wait_all(&acc_empty[ab], ((chain >> 1) - 1) & 1u, &abort_flag)) ||
            !mbar_wait_all(&y_full[s], (i / kYSlots) & 1u, &abort_flag) ||
            !mbar_wait_all(&b_full[b], (i / kBSlots) & 1u, &abort_flag)) {
          if (lane == 0) set_error(a.err, kErrMmaTimeout);
          abort_flag = 1;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t sy = smem_u32(smem + s * S::kYBytes), sb = smem_u32(b_area + b * S::kBBytes);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < kRows / 16; ++kk)
            umma_f16_pair(tmem_base + ab * NT, umma_desc(sy + kk * 2048, 64 * kRows * 2, 1024),
                          umma_desc(sb + kk * 2048, 64 * kRows * 2, 1024), idesc, (!first || kk > 0) ? 1u : 0u);
          umma_commit_pair(&done_bar[i % kDone]);
          if (i % kChain == kChain - 1 || i == nkb - 1) umma_commit_pair(&acc_full[ab]);
        }
        __syncwarp();
      }
    }
  } else if (warp == 2) {
    int issued = 0;
    for (int i = 0; i < nkb; ++i) {
      const int s = i % kQSlots;
      if (i >= kQSlots && !mbar_wait_all(&q_empty[s], ((i / kQSlots) & 1u) ^ 1u, &abort_flag)) {
        if (lane == 0) set_error(a.err, kErrMmaTimeout);
        abort_flag = 1;
        break;
      }
      if (elect_one()) {
        mbar_expect_tx(&q_full[s], S::kQBytes);
        tma_load_2d(q_area + s * S::kQBytes, &tmQ, &q_full[s], n0, row0(i));
      }
      __syncwarp();
      issued = i + 1;
    }
    if (abort_flag) {
      for (int i = issued > kQSlots ? issued - kQSlots : 0; i < issued; ++i) {
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(&q_full[i % kQSlots], (i / kQSlots) & 1u) && globaltimer_ns() - t0 < kWaitNs) {
        }
      }
    }
  } else if (warp < 3 + kBSlots * S::kTeamW) {
    // a team keeps to one operand slot; warp w of it converts rows 32 (w & 1) + lane, columns
    // 64 (w >> 1) .. + 63: two groups, one 64-column box of the operand
    const int b = (warp - 3) / S::kTeamW, w = (warp - 3) % S::kTeamW;
    const int k = (w & 1) * 32 + lane, box = w >> 1;
    uint8_t* out = b_area + b * S::kBBytes + box * (64 * kRows * 2) + k * 128;
    const uint32_t full = cluster_addr(&b_full[b], 0);
    const int g0 = n0 / 32 + 2 * box;
    uint32_t byte[kAhead][2];
    auto fetch = [&](int i, uint32_t (&to)[2]) {
      const int r = row0(i) + k;
      const uint8_t* e = a.q8.e + static_cast<int64_t>(r) * a.q8.lde + g0;
#pragma unroll
      for (int u = 0; u < 2; ++u) to[u] = (i < nkb && r < n && g0 + u < a.groups) ? __ldg(e + u) : 0u;
    };
#pragma unroll
    for (int p = 0; p < kAhead; ++p) fetch(b + kBSlots * p, byte[p]);
    for (int i = b; i < nkb; i += kBSlots) {
      const int r0 = row0(i), qs = i % kQSlots;
      // the products of block i - kBSlots are done, so block i - kQSlots was converted and
      // its codes had come: the next wait begins in their slot's next phase
      if ((i >= kBSlots && !products_done(i - kBSlots)) ||
          !mbar_wait_all(&q_full[qs], (i / kQSlots) & 1u, &abort_flag)) {
        if (lane == 0) set_error(a.err, kErrMmaTimeout);
        abort_flag = 1;
        break;
      }
      const uint8_t* row = q_area + qs * S::kQBytes + k * 128;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const __nv_bfloat162 scale = group8_scale_bf16(byte[0][u]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 c = *reinterpret_cast<const uint4*>(row + (((box * 4 + u * 2 + h) ^ (k & 7)) << 4));
          uint4 v0 = values8_bf16(c.x, c.y, scale), v1 = values8_bf16(c.z, c.w, scale);
          if (r0 + k >= n) v0 = v1 = make_uint4(0u, 0u, 0u, 0u);
          *reinterpret_cast<uint4*>(out + (((u * 4 + h * 2) ^ (k & 7)) << 4)) = v0;
          *reinterpret_cast<uint4*>(out + (((u * 4 + h * 2 + 1) ^ (k & 7)) << 4)) = v1;
        }
      }
      if (i == tail) {
        // dY's rows by plain loads (a warp eight pieces of 8 columns), zeros past the live
        // rows.  Its slot: block i - kYSlots is done, as it comes before i - kBSlots
        const __nv_bfloat16* y = a.dy + static_cast<int64_t>(r0 + k) * a.lddy + m0 + box * 64;
        uint8_t* sy = smem + (i % kYSlots) * S::kYBytes + box * (64 * kRows * 2) + k * 128;
        const int cols = a.M - m0 - box * 64;
#pragma unroll 1
        for (int p = 0; p < 8; ++p) {
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (r0 + k < n && 8 * p < cols) v = first_columns(*reinterpret_cast<const uint4*>(y + 8 * p), cols - 8 * p);
          *reinterpret_cast<uint4*>(sy + ((p ^ (k & 7)) << 4)) = v;
        }
      }
#pragma unroll
      for (int p = 0; p + 1 < kAhead; ++p)
#pragma unroll
        for (int u = 0; u < 2; ++u) byte[p][u] = byte[p + 1][u];
      fetch(i + kBSlots * kAhead, byte[kAhead - 1]);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&q_empty[qs]);
        mbar_arrive_cluster(full);
      }
    }
  } else {
    // epilogue: warp w drains TMEM lanes of its quarter into the CTA's partial tile, laid out
    // as in ckpt8_dw_kernel
    const int quarter = warp & 3;
    for (int chain = 0; chain * kChain < nkb; ++chain) {
      const int ab = chain & 1;
      if (!mbar_wait_all(&acc_full[ab], (chain >> 1) & 1u, &abort_flag)) {
        if (lane == 0) set_error(a.err, kErrMmaTimeout);
        abort_flag = 1;
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
      for (int c = 0; c < NT; c += 32) {
        float v[32];
        tmem_ld32(tmem_base + static_cast<uint32_t>(ab * NT + c) + (static_cast<uint32_t>(quarter * 32) << 16), v);
        float* p = part + (static_cast<int64_t>(c / 32) * 4 + quarter) * 1024 + lane * 4;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (chain == 0)
            *reinterpret_cast<float4*>(p + j * 128) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          else
            red_add_v4(p + j * 128, v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(cluster_addr(&acc_empty[ab], 0));
    }
  }
  __syncthreads();
  cluster_sync();  // neither CTA leaves while the other may still use its memory or barriers
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    tmem_dealloc_pair(tmem_base, 2 * NT);
  }
}

// gW (+)= the partial tiles of the splits.  A thread takes four columns of a row of a tile (in
// the partial tiles' own order) and a fourth of the splits, in order; the four shares are
// joined in order through shared memory.
__global__ void __launch_bounds__(256) ckpt8_dw_sum_kernel(Ckpt8DwArgs a, DwPlan plan) {
  GB_PDL_ENTRY();
  __shared__ float4 sh4[4][64];
  const int n = live_rows(a.n_ptr, a.cap);
  const int kb_total = (n + plan.rows - 1) / plan.rows;
  const int splits = kb_total > 0 ? shares(kb_total, plan.splits, plan.min_kb).splits : 0;
  const int tile_floats = 128 * plan.mt * plan.nt;
  const int tiles = plan.m_tiles * plan.n_tiles;
  const int x = threadIdx.x & 63, share = threadIdx.x >> 6;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 64 + x;  // the grid covers the tiles exactly
  const int tile = static_cast<int>(i / (tile_floats / 4));
  const int at = static_cast<int>(i % (tile_floats / 4)) * 4;
  const int per = (splits + 3) / 4, k1 = min(splits, (share + 1) * per);
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  const float* p = a.work + static_cast<int64_t>(tile) * tile_floats + at;
#pragma unroll 8
  for (int k = share * per; k < k1; ++k) {
    const float4 v = *reinterpret_cast<const float4*>(p + static_cast<int64_t>(k) * tiles * tile_floats);
    s.x += v.x;
    s.y += v.y;
    s.z += v.z;
    s.w += v.w;
  }
  sh4[share][x] = s;
  __syncthreads();
  if (share != 0) return;
#pragma unroll
  for (int q = 1; q < 4; ++q) {
    const float4 v = sh4[q][x];
    s.x += v.x;
    s.y += v.y;
    s.z += v.z;
    s.w += v.w;
  }
  // at = ((c / 32) * 4 + quarter) * 1024 + j * 128 + lane * 4, c the column over the accumulators
  const int lane = (at / 4) % 32, j = (at / 128) % 8, quarter = (at / 1024) % 4;
  const int c = (at / 4096) * 32 + j * 4;
  add_quad(a, (tile / plan.n_tiles) * 128 * plan.mt + (c / plan.nt) * 128 + quarter * 32 + lane,
           (tile % plan.n_tiles) * plan.nt + c % plan.nt, s);
}

// Tile and shares for M x N over cap rows on num_sms SMs.  The large tile (256 x 256) reads
// each operand least often and converts each code once per 256 columns of dY; it needs
// enough rows for every SM to get some 32 blocks of them.  With fewer rows the small tile
// spreads the same work over four times as many CTAs, and few rows are split over the CTAs
// of one cluster, which sum their partial tiles over distributed shared memory: no second
// kernel and no work area.
DwPlan plan_for(int M, int N, int cap, int num_sms) {
  DwPlan p;
  int64_t kb = ceil_div(std::max(cap, 1), BK);
  p.rows = BK;
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
  p.pair = p.mt == 2 && p.nt == 256;
  if (p.pair) {
    p.rows = PairSmem::kRows;
    p.min_kb = 8;
    kb = ceil_div(std::max(cap, 1), p.rows);
  }
  const int64_t tiles = static_cast<int64_t>(p.m_tiles) * p.n_tiles;
  // a split's only chain: its partial tile needs no earlier ones
  if (p.mt == 1 && p.nt == 128 && kb <= 8 * kClusterKb) {
    p.cluster = true;
    p.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(8, kb / p.min_kb)));
    return p;
  }
  const int64_t at_once = p.pair ? num_sms / 2 : num_sms;
  p.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(at_once / tiles, kb / p.min_kb)));
  return p;
}

CUtensorMap map_y(const Ckpt8DwArgs& a, const DwPlan& p, int rows, int blocks) {
  return p.y_blocks ? tensor_map_blocks(CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.dy, a.dy_rows, a.dy_cols, a.lddy, 64, rows,
                                        blocks)
                    : tensor_map_bf16(a.dy, a.dy_rows, a.dy_cols, a.lddy, rows);
}
CUtensorMap map_q(const Ckpt8DwArgs& a, int rows) {
  return tensor_map_u8(a.q8.q, a.q_rows, a.q_cols, a.q8.ldq, 128, rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int MT, int NT>
void launch_t(const Ckpt8DwArgs& a, DwPlan p, cudaStream_t stream) {
  using S = DSmem<MT, NT>;
  p.y_blocks = a.dy_cols % 64 == 0;
  p.q_blocks = NT > 128 && a.q_cols % 128 == 0;
  const CUtensorMap my = map_y(a, p, BK, 2 * MT);
  const CUtensorMap mq = p.q_blocks ? tensor_map_blocks(CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.q8.q, a.q_rows, a.q_cols,
                                                        a.q8.ldq, 128, BK, NT / 128)
                                    : map_q(a, BK);
  auto kern = ckpt8_dw_kernel<MT, NT>;
  set_smem(reinterpret_cast<const void*>(kern), S::kBytes);
  launch_cluster_k(kern, dim3(static_cast<unsigned>(p.m_tiles * p.n_tiles * p.splits)), dim3(kThreads),
                   p.cluster ? static_cast<unsigned>(p.splits) : 1u, S::kBytes, stream, my, mq, a, p);
  GB_LAUNCH_CHECK();
}

void launch_pair(const Ckpt8DwArgs& a, DwPlan p, cudaStream_t stream) {
  using S = PairSmem;
  const CUtensorMap my = tensor_map_bf16(a.dy, a.dy_rows, a.dy_cols, a.lddy, S::kRows), mq = map_q(a, S::kRows);
  set_smem(reinterpret_cast<const void*>(ckpt8_dw_pair_kernel), S::kBytes);
  launch_cluster_k(ckpt8_dw_pair_kernel, dim3(static_cast<unsigned>(p.m_tiles * p.n_tiles * p.splits * 2)),
                   dim3(S::kThreads), 2, S::kBytes, stream, my, mq, a, p);
  GB_LAUNCH_CHECK();
}

}  // namespace

int64_t ckpt8_dw_work_floats(int M, int N, int cap, int num_sms) {
  const DwPlan p = plan_for(M, N, cap, num_sms);
  return p.cluster ? 0 : static_cast<int64_t>(p.m_tiles) * p.n_tiles * p.splits * 128 * p.mt * p.nt;
}

void launch_ckpt8_dw(const Ckpt8DwArgs& a, int num_sms, cudaStream_t stream) {
  const DwPlan p = plan_for(a.M, a.N, a.cap, num_sms);
  if (p.pair)
    launch_pair(a, p, stream);
  else if (p.mt == 2)
    launch_t<2, 128>(a, p, stream);
  else
    p.nt == 256 ? launch_t<1, 256>(a, p, stream) : launch_t<1, 128>(a, p, stream);
  if (p.cluster) return;
  const int64_t threads = static_cast<int64_t>(p.m_tiles) * p.n_tiles * 128 * p.mt * p.nt / 4;
  launch_k(ckpt8_dw_sum_kernel, dim3(static_cast<unsigned>(threads / 64)), dim3(256), 0, stream, a, p);
  GB_LAUNCH_CHECK();
}

}  // namespace dev
}  // namespace grappa
