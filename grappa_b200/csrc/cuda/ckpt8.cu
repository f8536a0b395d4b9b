// Rows to 8 bits and back, and the activation backward from 8-bit or bf16 rows.
//
// All three are one pass over their rows with a few operations an element (the
// activation's slope: an exponential and a division), so HBM bounds them.  A lane takes
// eight or sixteen columns of a row, several loads in flight.
#include <algorithm>
#include <type_traits>

#include "ckpt8.cuh"
#include "grappa/rng.h"
#include "kernels.h"
#include "linear_act.cuh"
#include "tcgen05.cuh"

namespace grappa {
namespace dev {

namespace {

constexpr int kThreads = 256;
constexpr int kRowsC = 2;  // rows a thread of the load kernel has in flight
// pieces of 16 bytes that a thread of the store kernel has in flight, and its CTAs an SM:
// 139058 x 512 bf16 with 2 pieces and 4 / 6 CTAs 40.3 / 35.4 us (94 % of the copy's rate), with 4
// pieces 40.7 (sixteen neighbouring columns a lane took 41)
template <typename T>
constexpr int kInFlight = sizeof(T) == 2 ? 2 : 4;
constexpr int kStoreCtas = 6;

// LPR lanes x P pieces of 16 bytes cover a row (blockIdx.y the next of wide rows); pieces of a
// lane lie LPR apart, so that loads and code stores are whole lines, and a group's pieces in
// neighbouring lanes.
template <typename T>
constexpr int kPieceCols = 16 / sizeof(T);
template <typename T, int LPR, int P>
__global__ void __launch_bounds__(kThreads, kStoreCtas) ckpt8_store_kernel(Ckpt8Args a) {
  GB_PDL_ENTRY();
  constexpr int kTeams = kThreads / LPR, kCols = kPieceCols<T>, kGroup = 32 / kCols, R = kInFlight<T> / P;
  static_assert(LPR % kGroup == 0, "groups in neighbouring lanes");
  const int n = live_rows(a.n_ptr, a.cap);
  const int t = threadIdx.x % LPR, team = threadIdx.x / LPR;
  const int c0 = (blockIdx.y * P * LPR + t) * kCols;
  const int q_cols = (a.dim + 31) / 32 * 32;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kTeams * R; base < n;
       base += static_cast<int64_t>(gridDim.x) * kTeams * R) {
    uint4 raw[R][P];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * kTeams + team;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int c = c0 + i * LPR * kCols;
        raw[r][i] = row < n && c < a.dim
                        ? *reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + row * a.ld + c)
                        : make_uint4(0u, 0u, 0u, 0u);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * kTeams + team;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int c = c0 + i * LPR * kCols;
        if (c + kCols > a.dim) raw[r][i] = first_columns<T>(raw[r][i], a.dim - c);
        float v[8];
        float m;
        if constexpr (kCols == 8) {
          bf16x8_to_f32(raw[r][i], v);
          m = abs_max8(v);
        } else {
          v[0] = __uint_as_float(raw[r][i].x), v[1] = __uint_as_float(raw[r][i].y);
          v[2] = __uint_as_float(raw[r][i].z), v[3] = __uint_as_float(raw[r][i].w);
          m = max_nan(abs_max3(fabsf(v[0]), v[1], v[2]), fabsf(v[3]));
        }
#pragma unroll
        for (int o = 1; o < kGroup; o <<= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
        const uint32_t byte = group8_byte(m);
        const float inv = group8_inv(byte);
        if (row < n && c < q_cols) {
          int8_t* q = a.q8.q + row * a.q8.ldq + c;
          if constexpr (kCols == 8)
            *reinterpret_cast<uint2*>(q) = codes8(v, inv);
          else
            *reinterpret_cast<uint32_t*>(q) = codes4(v, inv);
          if (t % kGroup == 0) a.q8.e[row * a.q8.lde + (c >> 5)] = static_cast<uint8_t>(byte);
        }
      }
    }
  }
}

// LPR lanes x 16 columns cover a row; a lane's 16 columns are pieces of 16 output bytes LPR
// pieces apart, so that a store writes whole lines (sixteen neighbouring columns a lane, in
// half and quarter sectors: 65537 x 992 to fp32 80 us instead of 58, 139058 x 512 to bf16 38
// instead of 35: 94 % of the copy's rate)
template <typename T, int LPR>
__global__ void __launch_bounds__(kThreads, 4) ckpt8_load_kernel(Ckpt8Args a) {
  GB_PDL_ENTRY();
  constexpr int kTeams = kThreads / LPR;
  constexpr int kCols = 16 / sizeof(T), kPieces = 16 / kCols;
  const int n = live_rows(a.n_ptr, a.cap);
  const int t = threadIdx.x % LPR, team = threadIdx.x / LPR;
  const int c0 = blockIdx.y * LPR * 16 + t * kCols;
  const int cols = (a.dim + 7) / 8 * 8;  // zeros from dim on
  using Codes = std::conditional_t<kCols == 8, uint2, uint32_t>;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kTeams * kRowsC; base < n;
       base += static_cast<int64_t>(gridDim.x) * kTeams * kRowsC) {
    Codes q[kRowsC][kPieces];
    uint32_t e[kRowsC][kPieces];
#pragma unroll
    for (int r = 0; r < kRowsC; ++r) {
      const int64_t row = base + r * kTeams + team;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int c = c0 + i * LPR * kCols;
        q[r][i] = Codes();
        e[r][i] = 0u;
        if (row < n && c < cols) {
          q[r][i] = *reinterpret_cast<const Codes*>(a.q8.q + row * a.q8.ldq + c);
          e[r][i] = a.q8.e[row * a.q8.lde + (c >> 5)];
        }
      }
    }
#pragma unroll
    for (int r = 0; r < kRowsC; ++r) {
      const int64_t row = base + r * kTeams + team;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int c = c0 + i * LPR * kCols;
        if (row >= n || c >= cols) continue;
        uint4 o;
        if constexpr (kCols == 8) {
          o = values8_bf16(q[r][i].x, q[r][i].y, group8_scale_bf16(e[r][i]));
        } else {
          float v[4];
          values4(q[r][i], group8_scale(e[r][i]), v);
          o = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        }
        if (c + kCols > a.dim) o = first_columns<T>(o, a.dim - c);
        *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + row * a.ld + c) = o;
      }
    }
  }
}

template <typename T, int LPR, int P>
void store_t(const Ckpt8Args& a, cudaStream_t stream) {
  const int64_t passes = ceil_div(a.cap, kThreads / LPR * (kInFlight<T> / P));
  const int64_t slices = ceil_div(ceil_div(a.dim, 32) * 32, LPR * P * kPieceCols<T>);
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(passes, ceil_div(sm_count() * kStoreCtas, slices))),
                  static_cast<unsigned>(slices));
  launch_k(ckpt8_store_kernel<T, LPR, P>, grid, dim3(kThreads), 0, stream, a);
  GB_LAUNCH_CHECK();
}
template <typename T>
void store_rows(const Ckpt8Args& a, cudaStream_t stream) {
  constexpr int kCols = kPieceCols<T>;
  if (a.dim <= 32) return store_t<T, 32 / kCols, 1>(a, stream);
  if (a.dim <= 64) return store_t<T, 64 / kCols, 1>(a, stream);
  if (a.dim <= 128) return store_t<T, 128 / kCols, 1>(a, stream);
  if (a.dim <= 256) return store_t<T, 32, 8 / kCols>(a, stream);
  return store_t<T, 32, 16 / kCols>(a, stream);
}

// calls f with the lanes per row (a compile-time constant) for rows of `dim` columns
template <typename F>
void with_lpr(int dim, F&& f) {
  if (dim <= 32) return f(std::integral_constant<int, 2>());
  if (dim <= 64) return f(std::integral_constant<int, 4>());
  if (dim <= 128) return f(std::integral_constant<int, 8>());
  if (dim <= 256) return f(std::integral_constant<int, 16>());
  return f(std::integral_constant<int, 32>());
}
template <int LPR>
dim3 ckpt_grid(int dim, int cap) {
  // as many CTAs as the SMs hold at once: short-lived ones measured a third slower
  const int64_t passes = ceil_div(cap, kThreads / LPR * kRowsC), slices = ceil_div(ceil_div(dim, 32) * 2, LPR);
  return dim3(static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(passes, ceil_div(sm_count() * 4, slices)))),
              static_cast<unsigned>(slices));
}

// dz = mask(dout) act'(z): LPR lanes x 8 columns a row; blockIdx.y walks the 256-column slices
// of wide rows.  The column sums go through shared memory into one part a CTA, as in the
// norm's backward.  The next row is asked for as soon as
// this one is in fp32: 139058 x 256 from fp32 and 8-bit rows with GELU 45.3 -> 41.5 us (93 % of
// the copy's rate), 65536 x 1024 with SiLU 80 -> 74; from bf16 rows (45 -> 41) the slope's
// arithmetic bounds it.
template <int LPR, bool F32, bool Q8>
__global__ void __launch_bounds__(kThreads, 4) linear_act_bwd_kernel(LinearActBwdArgs a) {
  GB_PDL_ENTRY();
  constexpr int kTeams = kThreads / LPR;
  __shared__ float parts[kTeams][LPR * 8];
  const int t = threadIdx.x % LPR, team = threadIdx.x / LPR;
  const int n = live_rows(a.n_ptr, a.cap);
  const int n_end = min(a.cap, (n + 63) / 64 * 64);
  const int c = blockIdx.y * 32 + t;
  const bool col_on = c * 8 < a.dim;
  const uint64_t key = a.dropout_p > 0.f ? hop_key(static_cast<uint64_t>(a.counters[0]) ^ 0xD80Full,
                                                   static_cast<uint64_t>(a.counters[1]),
                                                   static_cast<uint64_t>(a.counters[2]), a.dropout_salt)
                                         : 0ull;
  const uint32_t thr8 = dropout_thr8(a.dropout_p);
  const float keep_scale = dropout_scale8(thr8);
  float acc[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = 0.f;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kTeams;
  uint4 g0, g1, zr;
  uint32_t eb;
  auto fetch = [&](int64_t row) {
    g0 = g1 = zr = make_uint4(0u, 0u, 0u, 0u);
    eb = 0;
    if (row >= n || !col_on) return;
    if constexpr (F32) {
      const uint4* p = reinterpret_cast<const uint4*>(static_cast<const float*>(a.dout) + row * a.lddo + c * 8);
      g0 = p[0];
      g1 = p[1];
    } else {
      g0 = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.dout) + row * a.lddo + c * 8);
    }
    if constexpr (Q8) {
      const uint2 q = *reinterpret_cast<const uint2*>(a.q8.q + row * a.q8.ldq + c * 8);
      zr = make_uint4(q.x, q.y, 0u, 0u);
      eb = a.q8.e[row * a.q8.lde + (c >> 2)];
    } else if (a.z) {
      zr = *reinterpret_cast<const uint4*>(a.z + row * a.ldz + c * 8);
    }
  };
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kTeams + team;
  fetch(row0);
  for (int64_t row = row0; row < n_end && col_on; row += step) {
    float g[8], z[8];
    if constexpr (F32) {
      const uint32_t w[8] = {g0.x, g0.y, g0.z, g0.w, g1.x, g1.y, g1.z, g1.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = __uint_as_float(w[j]);
    } else {
      bf16x8_to_f32(g0, g);
    }
    if constexpr (Q8)
      values8(make_uint2(zr.x, zr.y), group8_scale(eb), z);
    else
      bf16x8_to_f32(zr, z);
    fetch(row + step);
    if (c * 8 + 8 > a.dim) {
      mask8(g, c, a.dim);
      mask8(z, c, a.dim);
    }
    if (a.act == kActRelu) {
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = z[j] > 0.f ? g[j] : 0.f;
    } else if (a.act == kActGelu) {
#pragma unroll
      for (int j = 0; j < 8; j += 2) gelu_slope2(z + j, g + j);
    } else if (a.act == kActSilu) {
#pragma unroll
      for (int j = 0; j < 8; j += 2) silu_slope2(z + j, g + j);
    }
    if (a.dropout_p > 0.f) {
      const uint64_t at = static_cast<uint64_t>(row) * static_cast<uint64_t>(a.ld_mask) + static_cast<uint64_t>(c) * 8;
      const uint32_t keep = dropout_keep_bits(key, at, 8, thr8);
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = (keep >> j) & 1u ? g[j] * keep_scale : 0.f;
    }
    if (row < n) {
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] += g[j];
      if (a.clear_dout) {
        const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if constexpr (F32)
          store8(static_cast<float*>(a.dout) + row * a.lddo + c * 8, zero);
        else
          store8(static_cast<__nv_bfloat16*>(a.dout) + row * a.lddo + c * 8, zero);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] = 0.f;
    }
    store8(a.dz + row * a.lddz + c * 8, g);
  }
  if (!a.dbias) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) parts[team][t * 8 + j] = acc[j];
  __syncthreads();
  const int col0 = blockIdx.y * 256;
  float s = 0.f;
  if (threadIdx.x < LPR * 8) {
#pragma unroll 8
    for (int p = 0; p < kTeams; ++p) s += parts[p][threadIdx.x];
  }
  if (a.cluster) {
    // the slice's CTAs are one cluster, which finishes the sums
    __shared__ float cols[LPR * 8];
    if (threadIdx.x < LPR * 8) cols[threadIdx.x] = s;
    cluster_column_sums(cols, min(LPR * 8, a.dim - col0), a.dbias + col0, a.accumulate);
  } else if (threadIdx.x < LPR * 8 && col0 + static_cast<int>(threadIdx.x) < a.dim) {
    a.work[static_cast<int64_t>(blockIdx.x) * a.dim + col0 + threadIdx.x] = s;
  }
}

constexpr int kCtasPerSm = 4;

int64_t act_bwd_passes(int dim, int cap) {
  const int lpr = dim <= 32 ? 4 : dim <= 64 ? 8 : dim <= 128 ? 16 : 32;
  return ceil_div(std::max(cap, 1), kThreads / lpr);
}
int act_bwd_grid(int dim, int cap, int num_sms) {
  const int64_t slices = ceil_div(dim, 256);
  return static_cast<int>(std::max<int64_t>(
      1, std::min<int64_t>(act_bwd_passes(dim, cap), std::max<int64_t>(1, static_cast<int64_t>(num_sms) * kCtasPerSm / slices))));
}

template <int LPR>
void act_bwd_t(const LinearActBwdArgs& a, dim3 grid, cudaStream_t stream) {
  auto kern = a.dout_f32 ? (a.q8.q ? linear_act_bwd_kernel<LPR, true, true> : linear_act_bwd_kernel<LPR, true, false>)
                         : (a.q8.q ? linear_act_bwd_kernel<LPR, false, true> : linear_act_bwd_kernel<LPR, false, false>);
  launch_cluster_k(kern, grid, dim3(kThreads), a.cluster ? grid.x : 1u, 0, stream, a);
  GB_LAUNCH_CHECK();
}

}  // namespace

int64_t linear_act_bwd_work_floats(int dim, int cap, int num_sms) {
  return act_bwd_passes(dim, cap) <= kClusterPasses ? 0 : static_cast<int64_t>(dim) * act_bwd_grid(dim, cap, num_sms);
}

void launch_linear_act_bwd(LinearActBwdArgs a, int num_sms, cudaStream_t stream) {
  int gx = act_bwd_grid(a.dim, a.cap, num_sms);
  a.cluster = a.dbias && act_bwd_passes(a.dim, a.cap) <= kClusterPasses;
  if (a.cluster) gx = std::min(gx, 8);
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(ceil_div(a.dim, 256)));
  if (a.dim <= 32)
    act_bwd_t<4>(a, grid, stream);
  else if (a.dim <= 64)
    act_bwd_t<8>(a, grid, stream);
  else if (a.dim <= 128)
    act_bwd_t<16>(a, grid, stream);
  else
    act_bwd_t<32>(a, grid, stream);
  if (a.dbias && !a.cluster) launch_sum_parts(a.work, gx, a.dim, a.dim, a.dbias, a.accumulate, stream);
}

void launch_ckpt8_store(const Ckpt8Args& a, cudaStream_t stream) {
  if (a.cap <= 0) return;
  a.f32 ? store_rows<float>(a, stream) : store_rows<__nv_bfloat16>(a, stream);
}

void launch_ckpt8_load(const Ckpt8Args& a, cudaStream_t stream) {
  if (a.cap <= 0) return;
  with_lpr(a.dim, [&](auto lpr) {
    constexpr int L = decltype(lpr)::value;
    launch_k(a.f32 ? ckpt8_load_kernel<float, L> : ckpt8_load_kernel<__nv_bfloat16, L>, ckpt_grid<L>(a.dim, a.cap),
             dim3(kThreads), 0, stream, a);
  });
  GB_LAUNCH_CHECK();
}

}  // namespace dev
}  // namespace grappa
