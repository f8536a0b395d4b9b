// Rows to 8 bits and back, and the activation backward from 8-bit or bf16 rows.
//
// All three are one pass over their rows with a few operations an element (the
// activation's slope: an exponential and a division), so HBM bounds them.  A lane takes
// eight columns (16 bytes of bf16) of a row; four neighbouring lanes hold a group of 32
// and find its largest magnitude with two shuffles.
#include <algorithm>

#include "ckpt8.cuh"
#include "grappa/rng.h"
#include "kernels.h"
#include "linear_act.cuh"

namespace grappa {
namespace dev {

namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // chunks a thread has in flight

// A CTA takes kThreads * kUnroll chunks of consecutive rows; chunk i of the tile is column
// chunk i % cpr of row i / cpr (cpr: chunks of a row up to the next group, a multiple of 4,
// so a group never straddles two rows and its four chunks are four neighbouring lanes).
template <typename T>
__global__ void __launch_bounds__(kThreads) ckpt8_store_kernel(Ckpt8Args a) {
  GB_PDL_ENTRY();
  const int n = live_rows(a.n_ptr, a.cap);
  const uint32_t cpr = static_cast<uint32_t>((a.dim + 31) / 32 * 4);
  const int64_t total = static_cast<int64_t>(n) * cpr;
  const int64_t tile0 = static_cast<int64_t>(blockIdx.x) * (kThreads * kUnroll);
  if (tile0 >= total) return;
  const int64_t row0 = tile0 / cpr;
  const uint32_t off0 = static_cast<uint32_t>(tile0 - row0 * cpr);
  float v[kUnroll][8];
  int64_t row[kUnroll];
  uint32_t c[kUnroll];
  bool live[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t i = off0 + u * kThreads + threadIdx.x;
    row[u] = row0 + i / cpr;
    c[u] = i % cpr;
    live[u] = row[u] < n;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[u][j] = 0.f;
    if (live[u] && c[u] * 8 < static_cast<uint32_t>(a.dim)) load8(static_cast<const T*>(a.x) + row[u] * a.ld + c[u] * 8, v[u]);
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    mask8(v[u], static_cast<int>(c[u]), a.dim);
    uint32_t m = abs_max_bits8(v[u]);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const uint32_t byte = group8_byte(m);
    if (live[u]) {
      *reinterpret_cast<uint2*>(a.q8.q + row[u] * a.q8.ldq + c[u] * 8) = codes8(v[u], group8_inv(byte));
      if ((c[u] & 3u) == 0) a.q8.e[row[u] * a.q8.lde + (c[u] >> 2)] = static_cast<uint8_t>(byte);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) ckpt8_load_kernel(Ckpt8Args a) {
  GB_PDL_ENTRY();
  const int n = live_rows(a.n_ptr, a.cap);
  const uint32_t cpr = static_cast<uint32_t>((a.dim + 7) / 8);
  const int64_t total = static_cast<int64_t>(n) * cpr;
  const int64_t tile0 = static_cast<int64_t>(blockIdx.x) * (kThreads * kUnroll);
  if (tile0 >= total) return;
  const int64_t row0 = tile0 / cpr;
  const uint32_t off0 = static_cast<uint32_t>(tile0 - row0 * cpr);
  uint2 q[kUnroll];
  uint32_t e[kUnroll], c[kUnroll];
  int64_t row[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t i = off0 + u * kThreads + threadIdx.x;
    row[u] = row0 + i / cpr;
    c[u] = i % cpr;
    q[u] = make_uint2(0u, 0u);
    e[u] = 0;
    if (row[u] < n) {
      q[u] = *reinterpret_cast<const uint2*>(a.q8.q + row[u] * a.q8.ldq + c[u] * 8);
      e[u] = a.q8.e[row[u] * a.q8.lde + (c[u] >> 2)];
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    float v[8];
    values8(q[u], group8_scale(e[u]), v);
    mask8(v, static_cast<int>(c[u]), a.dim);
    if (row[u] < n) store8(static_cast<T*>(a.out) + row[u] * a.ld + c[u] * 8, v);
  }
}

// dz = mask(dout) act'(z): a warp takes LPR lanes x 8 columns of 32 / LPR rows, kRows of
// them in flight; blockIdx.y walks the 256-column slices of wide rows.  The column sums go
// through shared memory into one part a CTA, as in the norm's backward.
constexpr int kRows = 4;

template <int LPR, bool F32, bool Q8>
__global__ void __launch_bounds__(kThreads) linear_act_bwd_kernel(LinearActBwdArgs a) {
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
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kTeams * kRows; base < n_end;
       base += static_cast<int64_t>(gridDim.x) * kTeams * kRows) {
    uint4 g0[kRows], g1[kRows], zr[kRows];
    uint32_t eb[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int64_t row = base + r * kTeams + team;
      g0[r] = g1[r] = zr[r] = make_uint4(0u, 0u, 0u, 0u);
      eb[r] = 0;
      if (row < n && col_on) {
        if constexpr (F32) {
          const uint4* p = reinterpret_cast<const uint4*>(static_cast<const float*>(a.dout) + row * a.lddo + c * 8);
          g0[r] = p[0];
          g1[r] = p[1];
        } else {
          g0[r] = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.dout) + row * a.lddo + c * 8);
        }
        if constexpr (Q8) {
          const uint2 q = *reinterpret_cast<const uint2*>(a.q8.q + row * a.q8.ldq + c * 8);
          zr[r] = make_uint4(q.x, q.y, 0u, 0u);
          eb[r] = a.q8.e[row * a.q8.lde + (c >> 2)];
        } else if (a.z) {
          zr[r] = *reinterpret_cast<const uint4*>(a.z + row * a.ldz + c * 8);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int64_t row = base + r * kTeams + team;
      if (row >= n_end || !col_on) continue;
      float g[8], z[8];
      if constexpr (F32) {
        const uint32_t w[8] = {g0[r].x, g0[r].y, g0[r].z, g0[r].w, g1[r].x, g1[r].y, g1[r].z, g1[r].w};
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = __uint_as_float(w[j]);
      } else {
        bf16x8_to_f32(g0[r], g);
      }
      if constexpr (Q8)
        values8(make_uint2(zr[r].x, zr[r].y), group8_scale(eb[r]), z);
      else
        bf16x8_to_f32(zr[r], z);
      mask8(g, c, a.dim);
      mask8(z, c, a.dim);
      if (a.act == kActRelu) {
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = z[j] > 0.f ? g[j] : 0.f;
      } else if (a.act == kActGelu) {
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] *= gelu_slope(z[j]);
      } else if (a.act == kActSilu) {
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] *= silu_slope(z[j]);
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
  }
  if (!a.dbias) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) parts[team][t * 8 + j] = acc[j];
  __syncthreads();
  const int col = blockIdx.y * 256 + threadIdx.x;
  if (threadIdx.x < LPR * 8 && col < a.dim) {
    float s = 0.f;
#pragma unroll 8
    for (int p = 0; p < kTeams; ++p) s += parts[p][threadIdx.x];
    a.work[static_cast<int64_t>(blockIdx.x) * a.dim + col] = s;
  }
}

constexpr int kCtasPerSm = 8;

int act_bwd_grid(int dim, int cap, int num_sms) {
  const int lpr = dim <= 32 ? 4 : dim <= 64 ? 8 : dim <= 128 ? 16 : 32;
  const int64_t slices = ceil_div(dim, 256);
  const int64_t want = ceil_div(std::max(cap, 1), kThreads / lpr * kRows);
  return static_cast<int>(std::max<int64_t>(
      1, std::min<int64_t>(want, std::max<int64_t>(1, static_cast<int64_t>(num_sms) * kCtasPerSm / slices))));
}

template <int LPR>
void act_bwd_t(const LinearActBwdArgs& a, dim3 grid, cudaStream_t stream) {
  auto kern = a.dout_f32 ? (a.q8.q ? linear_act_bwd_kernel<LPR, true, true> : linear_act_bwd_kernel<LPR, true, false>)
                         : (a.q8.q ? linear_act_bwd_kernel<LPR, false, true> : linear_act_bwd_kernel<LPR, false, false>);
  launch_k(kern, grid, dim3(kThreads), 0, stream, a);
  GB_LAUNCH_CHECK();
}

}  // namespace

int64_t linear_act_bwd_work_floats(int dim, int cap, int num_sms) {
  return static_cast<int64_t>(dim) * act_bwd_grid(dim, cap, num_sms);
}

void launch_linear_act_bwd(const LinearActBwdArgs& a, int num_sms, cudaStream_t stream) {
  const int gx = act_bwd_grid(a.dim, a.cap, num_sms);
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(ceil_div(a.dim, 256)));
  if (a.dim <= 32)
    act_bwd_t<4>(a, grid, stream);
  else if (a.dim <= 64)
    act_bwd_t<8>(a, grid, stream);
  else if (a.dim <= 128)
    act_bwd_t<16>(a, grid, stream);
  else
    act_bwd_t<32>(a, grid, stream);
  if (a.dbias) launch_sum_parts(a.work, gx, a.dim, a.dim, a.dbias, a.accumulate, stream);
}

void launch_ckpt8_store(const Ckpt8Args& a, cudaStream_t stream) {
  if (a.cap <= 0) return;
  const int64_t grid = ceil_div(static_cast<int64_t>(a.cap) * ceil_div(a.dim, 32) * 4, kThreads * kUnroll);
  launch_k(a.f32 ? ckpt8_store_kernel<float> : ckpt8_store_kernel<__nv_bfloat16>, dim3(static_cast<unsigned>(grid)),
           dim3(kThreads), 0, stream, a);
  GB_LAUNCH_CHECK();
}

void launch_ckpt8_load(const Ckpt8Args& a, cudaStream_t stream) {
  if (a.cap <= 0) return;
  const int64_t grid = ceil_div(static_cast<int64_t>(a.cap) * ceil_div(a.dim, 8), kThreads * kUnroll);
  launch_k(a.f32 ? ckpt8_load_kernel<float> : ckpt8_load_kernel<__nv_bfloat16>, dim3(static_cast<unsigned>(grid)),
           dim3(kThreads), 0, stream, a);
  GB_LAUNCH_CHECK();
}

}  // namespace dev
}  // namespace grappa
