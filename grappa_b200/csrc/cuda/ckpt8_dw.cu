// Weight gradient from rows kept in 8 bits: gW[M][N] (+)= dY^T Xh, Xh the rows that the
// codes stand for, exact in bf16.  The reduction runs over the rows, so both operands are
// MN-major and read in place.
//
// A tile is 128 x 128 outputs of one CTA, or 256 x 256 of a CTA pair (cta_group::2): each CTA
// of the pair loads 128 columns of dY and of codes, converts its own, and the products read
// both CTAs' operands, which halves the operand bytes that an SM's tensor core reads.  A CTA
// walks its share of the rows, 64 at a time:
//   warp 0        TMA producer of dY, on CTA 0's barrier, straight into the MMA's layout
//   warp 1        (CTA 0) issues the products
//   warp 2        TMA producer of the codes, on the CTA's own barriers
//   warps 3..18   turn codes into the bf16 operand, four warps a block (32 rows x 64 columns
//                 each), one team of them for every operand slot
//   warps 19..22  empty the accumulator: there are two, so that the products of the next 2048
//                 rows run meanwhile
// dY, codes and converted rows have rings of their own, each as long as its way round wants:
// dY is held from its load to the end of its products, the codes until they are converted, the
// operand from there to the end of the products.  One commit a block says that its products
// are done.  The last block of a partly filled 64 rows takes its dY through the converters,
// which write zeros for the rows past the live ones.
//
// What bounds it: the bf16 form of the rows never leaves the SM; HBM sees dY once and 33/32
// bytes a kept value.  500009 x 512 x 256 (kept columns x dY's) takes 141 us, where HBM wants
// 81 and the products 78.  A pair spends some 1200 cycles on a block whose products take 640:
// the loads alone took 103 us, and conversion, loads and the products' operand reads share
// the SM's shared memory.
//
// Accuracy: the tensor core adds into its fp32 accumulator by truncation, so a sum over R
// rows drifts by about 1.2e-9 R of itself (measured on the bf16 GEMM: 1.6e-4 at 139058 rows,
// 4e-6 at 3758).  The accumulator is therefore emptied every kChainRows rows into the CTA's
// own partial tile, in fp32 with rounding to nearest (the first time a store, then reductions
// that this thread alone makes to these addresses, so their order is fixed).  A second kernel,
// or the splits of a tile as one cluster, adds the partial tiles in order: the same bits every
// time.
#include <algorithm>

#include "ckpt8.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

namespace grappa {
namespace dev {

namespace {

constexpr int kChainRows = 2048;
constexpr int kAhead = 2;          // own blocks whose exponents are asked for ahead
constexpr int kSplitsCluster = 8;  // splits that a cluster holds

// Shared memory and warps; CG the CTAs of a tile.
template <int CG>
struct DwSmem {
  static constexpr int kRows = 64;
  static constexpr int kYBytes = 128 * kRows * 2, kYSlots = 7;
  static constexpr int kBBytes = 128 * kRows * 2, kBSlots = 4;
  static constexpr int kQBytes = 128 * kRows, kQSlots = 5;
  static constexpr int kDone = 8;                            // barriers of finished blocks
  static constexpr int kTeamW = 4;                           // warps of a team
  static constexpr int kWarps = 3 + kBSlots * kTeamW + 4;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kChain = kChainRows / kRows;
  static constexpr int NT = 128 * CG;                        // columns of the tile
  static constexpr int kBytes = kYSlots * kYBytes + kBSlots * kBBytes + kQSlots * kQBytes + 1024 /*align*/;
  static_assert(kBytes <= 226 * 1024 && kDone >= kYSlots && kQSlots > kBSlots, "ckpt8_dw: shared memory");
};
constexpr int kRows = DwSmem<1>::kRows;

// How the rows are shared: kb_total blocks of kRows rows over `splits` CTAs a tile, fewer
// when the live rows are few (each then takes at least min_kb blocks, or one takes all).
__device__ __forceinline__ int live_splits(int kb_total, int splits_max, int min_kb) {
  return max(1, min(splits_max, kb_total / min_kb));
}

struct DwPlan {
  int cg;                // CTAs of a tile, which has 128 cg x 128 cg outputs
  int m_tiles, n_tiles;
  int splits, min_kb;    // shares of the rows at most, blocks each at least
  bool cluster;          // a tile's splits are one cluster that sums its partial tiles itself
};

// The first `cols` of eight columns at p, zeros after them.  A row may end with its M columns,
// so a piece that is not whole is read column by column.
__device__ __forceinline__ uint4 row_piece(const __nv_bfloat16* p, int cols) {
  if (cols >= 8) return *reinterpret_cast<const uint4*>(p);
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < 7; ++j)
    if (j < cols) w[j >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[j]) << (16 * (j & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

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

template <int CG>
__global__ void __launch_bounds__(DwSmem<CG>::kThreads, 1)
    ckpt8_dw_kernel(const __grid_constant__ CUtensorMap tmY, const __grid_constant__ CUtensorMap tmQ, Ckpt8DwArgs a,
                    DwPlan plan) {
  using S = DwSmem<CG>;
  constexpr int kYSlots = S::kYSlots, kBSlots = S::kBSlots, kQSlots = S::kQSlots, kDone = S::kDone;
  constexpr int kChain = S::kChain, NT = S::NT;
  const bool cluster = CG == 1 && plan.cluster;
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
    for (int s = 0; s < kBSlots; ++s) mbar_init(&b_full[s], CG * S::kTeamW);  // the block's team in every CTA
    for (int s = 0; s < kQSlots; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], S::kTeamW);
    }
    for (int s = 0; s < kDone; ++s) mbar_init(&done_bar[s], 1);
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], CG * 4);  // four warps in every CTA
    }
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_map(&tmY);
    prefetch_map(&tmQ);
  }
  if (warp == 1) CG == 2 ? tmem_alloc_pair(&tmem_slot, 2 * NT) : tmem_alloc(&tmem_slot, 2 * NT);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = tmem_slot;

  // all of this may run while the kernel before is ending; its results are read from here on
  GB_PDL_ENTRY();
  const int n = live_rows(a.n_ptr, a.cap);
  const int kb_total = (n + kRows - 1) / kRows;
  const int splits = live_splits(kb_total, plan.splits, plan.min_kb);
  const int tiles = plan.m_tiles * plan.n_tiles, unit = blockIdx.x / CG;
  const int rank = CG == 2 ? static_cast<int>(cluster_rank()) : 0;
  // the splits of a tile are a cluster, or tiles apart
  const int tile = cluster ? unit / plan.splits : unit % tiles;
  const int split = cluster ? unit % plan.splits : unit / tiles;
  const int m_tile = tile / plan.n_tiles;
  const int m0 = m_tile * NT + rank * 128, n0 = (tile - m_tile * plan.n_tiles) * NT + rank * 128;
  // the splits take the blocks in turn, so that the whole device reads one stretch of rows
  const int nkb = split < splits && kb_total > split ? (kb_total - split + splits - 1) / splits : 0;
  auto row0 = [&](int i) { return (split + i * splits) * kRows; };
  // number of the partly filled block (-1: none here)
  const int tail = n % kRows != 0 && nkb > 0 && row0(nkb - 1) + kRows > n ? nkb - 1 : -1;
  float* part = a.work + static_cast<int64_t>(blockIdx.x) * (128 * NT);
  // a wait for arrivals of both CTAs
  auto wait_both = [&](uint64_t* bar, uint32_t parity) {
    if constexpr (CG == 2) return mbar_wait_cluster(bar, parity, &abort_flag);
    return mbar_wait_all(bar, parity, &abort_flag);
  };
  // waits until the products of block j are done (j in order for every caller,
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
          if (rank == 0) mbar_expect_tx(&y_full[s], CG * S::kYBytes);
#pragma unroll
          for (int c = 0; c < 128; c += 64) {
            if constexpr (CG == 2)
              tma_load_2d_pair(sy + c * (kRows * 2), &tmY, cluster_addr(&y_full[s], 0), m0 + c, r0);
            else
              tma_load_2d(sy + c * (kRows * 2), &tmY, &y_full[s], m0 + c, r0);
          }
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
      constexpr uint32_t idesc = umma_idesc(128 * CG, NT, true, true);
      for (int i = 0; i < nkb; ++i) {
        const int s = i % kYSlots, b = i % kBSlots;
        const int chain = i / kChain, ab = chain & 1;
        const bool first = i % kChain == 0;
        if ((first && chain >= 2 && !wait_both(&acc_empty[ab], ((chain >> 1) - 1) & 1u)) ||
            !mbar_wait_all(&y_full[s], (i / kYSlots) & 1u, &abort_flag) ||
            !wait_both(&b_full[b], (i / kBSlots) & 1u)) {
          if (lane == 0) set_error(a.err, kErrMmaTimeout);
          abort_flag = 1;
          break;
        }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t sy = smem_u32(smem + s * S::kYBytes), sb = smem_u32(b_area + b * S::kBBytes);
        if (elect_one()) {
#pragma unroll
          for (int kk = 0; kk < kRows / 16; ++kk) {
            const uint64_t dy = umma_desc(sy + kk * 2048, 64 * kRows * 2, 1024);
            const uint64_t db = umma_desc(sb + kk * 2048, 64 * kRows * 2, 1024);
            const uint32_t add = (!first || kk > 0) ? 1u : 0u;
            if constexpr (CG == 2)
              umma_f16_pair(tmem_base + ab * NT, dy, db, idesc, add);
            else
              umma_f16(tmem_base + ab * NT, dy, db, idesc, add);
          }
          const bool last = i % kChain == kChain - 1 || i == nkb - 1;
          if constexpr (CG == 2) {
            umma_commit_pair(&done_bar[i % kDone]);
            if (last) umma_commit_pair(&acc_full[ab]);
          } else {
            umma_commit(&done_bar[i % kDone]);
            if (last) umma_commit(&acc_full[ab]);
          }
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
          if (r0 + k < n && 8 * p < cols) v = row_piece(y + 8 * p, cols - 8 * p);
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
        if constexpr (CG == 2)
          mbar_arrive_cluster(cluster_addr(&b_full[b], 0));
        else
          mbar_arrive(&b_full[b]);
      }
    }
  } else {
    // epilogue: a warp drains the TMEM lanes of its quarter into the CTA's partial tile, which
    // is laid out as the warp writes it: 32 columns at a time, 4 of them a lane and store, 512
    // bytes a store
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
        if (cluster) {
          // kept in the CTA's own shared memory, where the ring was (the only chain is over, so
          // every load and product of the ring is), row by row, pieces of 4 columns swizzled
          float4* t = reinterpret_cast<float4*>(smem) + (quarter * 32 + lane) * 32;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            t[(c / 4 + j) ^ lane] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          continue;
        }
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
      if (lane == 0) {
        if constexpr (CG == 2)
          mbar_arrive_cluster(cluster_addr(&acc_empty[ab], 0));
        else
          mbar_arrive(&acc_empty[ab]);
      }
    }
  }
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();  // neither CTA leaves while the other may use its memory or barriers
  if (cluster) {
    // gW (+)= the cluster's partial tiles, in order, each CTA a share of the tile
    // (a warp 128 columns of a row: whole lines of gW)
    cluster_sync();
    const int parts = kb_total > 0 ? splits : 0;
    for (int x = split * S::kThreads + static_cast<int>(threadIdx.x); x < 128 * 32; x += plan.splits * S::kThreads) {
      const int row = x / 32, k = x % 32;
      const uint8_t* at = smem + (row * 32 + (k ^ (row & 31))) * 16;
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
      float4 v[kSplitsCluster];
#pragma unroll
      for (int r = 0; r < kSplitsCluster; ++r) {
        v[r] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < parts) v[r] = ld_cluster4(cluster_addr(at, static_cast<uint32_t>(r)));
      }
#pragma unroll
      for (int r = 0; r < kSplitsCluster; ++r) s.x += v[r].x, s.y += v[r].y, s.z += v[r].z, s.w += v[r].w;
      add_quad(a, m0 + row, n0 + k * 4, s);
    }
    cluster_sync();  // the others may still read this CTA's tile
  }
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    CG == 2 ? tmem_dealloc_pair(tmem_base, 2 * NT) : tmem_dealloc(tmem_base, 2 * NT);
  }
}

// gW (+)= the partial tiles of the splits.  A thread takes four columns of a row of a tile (in
// the partial tiles' own order) and a fourth of the splits, in order; the four shares are
// joined in order through shared memory.
__global__ void __launch_bounds__(256) ckpt8_dw_sum_kernel(Ckpt8DwArgs a, DwPlan plan) {
  GB_PDL_ENTRY();
  __shared__ float4 sh4[4][64];
  const int n = live_rows(a.n_ptr, a.cap);
  const int kb_total = (n + kRows - 1) / kRows;
  const int splits = kb_total > 0 ? live_splits(kb_total, plan.splits, plan.min_kb) : 0;
  const int nt = 128 * plan.cg, tile_floats = nt * nt;
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
  // at = ((c / 32) * 4 + quarter) * 1024 + j * 128 + lane * 4, c the column over the CTAs' accumulators
  const int lane = (at / 4) % 32, j = (at / 128) % 8, quarter = (at / 1024) % 4;
  const int c = (at / 4096) * 32 + j * 4;
  add_quad(a, (tile / plan.n_tiles) * nt + (c / nt) * 128 + quarter * 32 + lane,
           (tile % plan.n_tiles) * nt + c % nt, s);
}

// Tile and shares for M x N over cap rows on num_sms SMs.  Measured, us, pairs / single CTAs:
// 8000 x 512 x 256 14.4 / 13.0, 12000 x 512 x 256 15.9 / 15.8, 20000 x 512 x 256 17.8 / 19.7,
// 50000 x 512 x 256 25.4 / 35.1, 5000 x 1024 x 1024 28 / 38: pairs from three blocks of their
// tiles an SM on, where more than 128 columns fill them (100000 x 256 x 128 25.2 / 23.0,
// 500009 x 128 x 128 71 / 46).
// Few rows: a cluster of single CTAs needs no second kernel and no work area, but is eight CTAs
// a tile at most.  Cluster / two kernels: 256 x 512 x 256 9.0 / 10.6, 1024 x 512 x 256
// 9.6 / 10.7, 2000 x 512 x 256 11.1 / 10.3 (and a launch less on the host), 3250 x 512 x 256
// 13.1 / 11.6, 12000 x 512 x 256 23 / 15.8.
// Blocks a share at least (4 / 8): pairs 6000 x 512 x 256 14.8 / 16.0, single CTAs 3250 x 512 x
// 256 11.6 / 13.5; 2 in a cluster (2 / 4: 256 rows 9.0 / 10.6, 1024 rows 9.6 / 10.3).
DwPlan plan_for(int M, int N, int cap, int num_sms) {
  DwPlan p;
  const int64_t kb = ceil_div(std::max(cap, 1), kRows);
  p.cg = M > 128 && N > 128 && ceil_div(M, 256) * ceil_div(N, 256) * kb >= 3ll * num_sms ? 2 : 1;
  constexpr int kClusterKb = 4 * kSplitsCluster;
  static_assert(kClusterKb <= DwSmem<1>::kChain, "a cluster's CTA has one chain");
  p.cluster = p.cg == 1 && kb <= kClusterKb;
  p.min_kb = p.cluster ? 2 : 4;
  p.m_tiles = static_cast<int>(ceil_div(M, 128 * p.cg));
  p.n_tiles = static_cast<int>(ceil_div(N, 128 * p.cg));
  const int64_t tiles = static_cast<int64_t>(p.m_tiles) * p.n_tiles;
  const int64_t most = p.cluster ? kSplitsCluster : num_sms / p.cg / tiles;
  p.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(most, kb / p.min_kb)));
  return p;
}

template <int CG>
void launch_t(const Ckpt8DwArgs& a, const DwPlan& p, cudaStream_t stream) {
  using S = DwSmem<CG>;
  const CUtensorMap my = tensor_map_bf16(a.dy, a.dy_rows, a.dy_cols, a.lddy, kRows);
  const CUtensorMap mq = tensor_map_u8(a.q8.q, a.q_rows, a.q_cols, a.q8.ldq, 128, kRows, CU_TENSOR_MAP_SWIZZLE_128B);
  auto kern = ckpt8_dw_kernel<CG>;
  set_smem(reinterpret_cast<const void*>(kern), S::kBytes);
  launch_cluster_k(kern, dim3(static_cast<unsigned>(p.m_tiles * p.n_tiles * p.splits * CG)), dim3(S::kThreads),
                   p.cluster ? static_cast<unsigned>(p.splits) : CG, S::kBytes, stream, my, mq, a, p);
  GB_LAUNCH_CHECK();
}

}  // namespace

int64_t ckpt8_dw_work_floats(int M, int N, int cap, int num_sms) {
  const DwPlan p = plan_for(M, N, cap, num_sms);
  return p.cluster ? 0 : static_cast<int64_t>(p.m_tiles) * p.n_tiles * p.splits * p.cg * p.cg * 16384;
}

void launch_ckpt8_dw(const Ckpt8DwArgs& a, int num_sms, cudaStream_t stream) {
  const DwPlan p = plan_for(a.M, a.N, a.cap, num_sms);
  p.cg == 2 ? launch_t<2>(a, p, stream) : launch_t<1>(a, p, stream);
  if (p.cluster) return;
  const int64_t threads = static_cast<int64_t>(p.m_tiles) * p.n_tiles * p.cg * p.cg * 4096;
  launch_k(ckpt8_dw_sum_kernel, dim3(static_cast<unsigned>(threads / 64)), dim3(256), 0, stream, a, p);
  GB_LAUNCH_CHECK();
}

}  // namespace dev
}  // namespace grappa
