// RMS norm of rows with the residual's addition, and its backward.
//
//   forward   s = x + r (rounded to the rows' type where it is written: the backward
//             pass reads those rows), rstd = 1 / sqrt(mean_j s_j^2 + eps),
//             y_j = s_j rstd gamma_j, and optionally xh_j = s_j rstd in 8 bits
//   backward  dx_j = rstd (gamma_j dy_j - xh_j c) + dr_j,  c = mean_j gamma_j dy_j xh_j,
//             dgamma_j = sum over the rows of dy_j xh_j
//
// Each row is read once and each output written once; a dozen operations an element, so
// HBM bounds both.  A team of lanes holds a row in registers, eight columns (one or two
// 16-byte loads) a lane: 4 to 32 lanes for rows of up to 256 columns, two to eight warps up to
// 2048, a whole CTA with two or four steps above.  Loads are kept in flight by two rows at a
// time (forward) or by asking for the next row early (backward).  The row sums are shuffles,
// and one shared-memory exchange for teams of several warps.  All sums and statistics are fp32.
// Measured: forward 139058 x 256 bf16 with residual and 8-bit rows 52.7 us, 94 % of the copy's
// rate; backward 1000003 x 128 from 8-bit rows 155 us, 90 %; 139058 x 256 bf16 49 us, 90 %.
//
// dgamma: a lane sums its columns over the rows of its team, the CTA joins its teams in
// shared memory in a fixed order and writes one part, and a second kernel sums the parts
// in order (a single cluster of CTAs, where the rows are few, joins them itself): the same
// bits every time, and no atomics.
#include <algorithm>

#include "ckpt8.cuh"
#include "kernels.h"

namespace grappa {
namespace dev {

namespace {

constexpr int kThreads = 256;

// Eight columns of a row as they lie in memory, so that every load of a step is issued
// before the first conversion.  Kinds: bf16, fp32, codes.
enum Kind : int { kBf = 0, kF32 = 1, kQ8 = 2 };
template <int K>
struct Raw8 {
  uint32_t w[K == kF32 ? 8 : (K == kBf ? 4 : 2)];
};
template <int K>
__device__ __forceinline__ Raw8<K> raw_zero() {
  Raw8<K> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(r.w) / 4); ++i) r.w[i] = 0u;
  return r;
}
template <int K>
__device__ __forceinline__ Raw8<K> raw_load(const void* base, int64_t at) {
  Raw8<K> r;
  if constexpr (K == kQ8) {
    const uint2 q = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(base) + at);
    r.w[0] = q.x, r.w[1] = q.y;
  } else if constexpr (K == kF32) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const float*>(base) + at);
    const uint4 a = p[0], b = p[1];
    r.w[0] = a.x, r.w[1] = a.y, r.w[2] = a.z, r.w[3] = a.w;
    r.w[4] = b.x, r.w[5] = b.y, r.w[6] = b.z, r.w[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(base) + at);
    r.w[0] = a.x, r.w[1] = a.y, r.w[2] = a.z, r.w[3] = a.w;
  }
  return r;
}
template <int K>
__device__ __forceinline__ void raw_values(const Raw8<K>& r, float scale, float* v) {
  if constexpr (K == kQ8) {
    values8(make_uint2(r.w[0], r.w[1]), scale, v);
  } else if constexpr (K == kF32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r.w[i]);
  } else {
    bf16x8_to_f32(make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]), v);
  }
}
template <int K>
__device__ __forceinline__ void store_kind(void* base, int64_t at, const float* v) {
  if constexpr (K == kF32)
    store8(static_cast<float*>(base) + at, v);
  else
    store8(static_cast<__nv_bfloat16*>(base) + at, v);
}

// sum over the team of R values a lane; teams of several warps exchange through sh[R][8]
template <int TEAM, int R>
__device__ __forceinline__ void team_sum(float (&s)[R], float (*sh)[8]) {
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int o = (TEAM < 32 ? TEAM : 32) / 2; o > 0; o >>= 1) s[r] += __shfl_xor_sync(0xffffffffu, s[r], o);
  }
  if constexpr (TEAM > 32) {
    constexpr int kWarps = TEAM / 32;
    const int w = threadIdx.x >> 5, w0 = w / kWarps * kWarps;
    __syncthreads();  // the last exchange has been read
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int r = 0; r < R; ++r) sh[r][w] = s[r];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s[r] = 0.f;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) s[r] += sh[r][w0 + i];
    }
  }
}

template <int K, int TEAM, int NV, int R>
__global__ void __launch_bounds__(kThreads, NV * R <= 2 ? 4 : 2) rmsnorm_fwd_kernel(RmsNormArgs a) {
  GB_PDL_ENTRY();
  __shared__ float sh[R][8];
  constexpr int kTeams = kThreads / TEAM;
  const int t = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
  const int n = live_rows(a.n_ptr, a.cap);
  const int chunks = (a.dim + 7) / 8;
  const int qchunks = a.q8.q ? (a.dim + 31) / 32 * 4 : chunks;
  const float inv_dim = 1.f / static_cast<float>(a.dim);
  float gam[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) gam[i][j] = (i * TEAM + t) * 8 + j < a.dim ? __ldg(a.gamma + (i * TEAM + t) * 8 + j) : 0.f;
  // a CTA takes kTeams * R consecutive rows at a time (uniform trip count per warp)
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * kTeams * R; base < n;
       base += static_cast<int64_t>(gridDim.x) * kTeams * R) {
    Raw8<K> raw[R][NV], rr[R][NV];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * kTeams + team;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = i * TEAM + t;
        const bool on = row < n && c < chunks;
        raw[r][i] = on ? raw_load<K>(a.x, row * a.ldx + c * 8) : raw_zero<K>();
        rr[r][i] = on && a.residual ? raw_load<K>(a.residual, row * a.ldr + c * 8) : raw_zero<K>();
      }
    }
    float v[R][NV][8], ss[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * kTeams + team;
      ss[r] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = i * TEAM + t;
        raw_values<K>(raw[r][i], 0.f, v[r][i]);
        if (a.residual) {
          float w[8];
          raw_values<K>(rr[r][i], 0.f, w);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[r][i][j] += w[j];
          if constexpr (K == kBf) bf16x8_to_f32(f32_to_bf16x8(v[r][i]), v[r][i]);
        }
        mask8(v[r][i], c, a.dim);
        if (a.s_out && row < n && c < chunks) store_kind<K>(a.s_out, row * a.lds + c * 8, v[r][i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) ss[r] = fmaf(v[r][i][j] * inv_dim, v[r][i][j], ss[r]);
      }
    }
    team_sum<TEAM, R>(ss, sh);  // the mean: each term is divided, so that it fits fp32 where the mean does
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * kTeams + team;
      const float rs = rsqrtf(ss[r] + a.eps);
      if (t == 0 && row < n) a.rstd[row] = rs;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = i * TEAM + t;
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[r][i][j] *= rs;
          y[j] = v[r][i][j] * gam[i][j];
        }
        if (row < n && c < chunks) {
          mask8(y, c, a.dim);  // an infinite or NaN row: its pad columns stay zero
          store8(a.y + row * a.ldy + c * 8, y);
        }
        if (a.q8.q) {
          float m = abs_max8(v[r][i]);
          m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
          m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 2));
          const uint32_t byte = group8_byte(m);
          if (row < n && c < qchunks) {
            *reinterpret_cast<uint2*>(a.q8.q + row * a.q8.ldq + c * 8) = codes8(v[r][i], group8_inv(byte));
            if ((c & 3) == 0) a.q8.e[row * a.q8.lde + (c >> 2)] = static_cast<uint8_t>(byte);
          }
        }
      }
    }
  }
}

// CTAs of the backward kernel that an SM holds
constexpr int bwd_ctas(int ky, int kx, int kd, int nv) {
  return nv > 1 ? 1 : (ky == kF32 || kx == kF32 || kd == kF32 ? 3 : 4);
}

template <int KY, int KX, int KD, int TEAM, int NV, int R>
__global__ void __launch_bounds__(kThreads, bwd_ctas(KY, KX, KD, NV))
    rmsnorm_bwd_kernel(RmsNormBwdArgs a) {
  GB_PDL_ENTRY();
  __shared__ float sh[R][8];
  extern __shared__ float parts[];  // [kTeams][TEAM * NV * 8] (several teams), then the column sums
  constexpr int kTeams = kThreads / TEAM;
  constexpr int kCols = TEAM * NV * 8;
  const int t = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
  const int n = live_rows(a.n_ptr, a.cap);
  const int n_res = a.dres ? min(live_rows(a.n_res_ptr, a.res_cap), n) : 0;
  const int chunks = (a.dim + 7) / 8;
  const float inv_dim = 1.f / static_cast<float>(a.dim);
  float acc[NV][8], gam[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int col = (i * TEAM + t) * 8 + j;
      acc[i][j] = 0.f;
      gam[i][j] = col < a.dim ? a.gamma[col] : 0.f;
    }
  }
  const int64_t step = static_cast<int64_t>(gridDim.x) * kTeams * R;
  Raw8<KY> yr[R][NV];
  Raw8<KX> xr[R][NV];
  Raw8<KD> rr[R][NV];
  uint32_t eb[R][NV];
  float rs_next[R];
  auto fetch = [&](int64_t base) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * kTeams + team;
      rs_next[r] = row < n ? a.rstd[row] : 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = i * TEAM + t;
        const bool on = row < n && c < chunks;
        yr[r][i] = on ? raw_load<KY>(a.dy, row * a.lddy + c * 8) : raw_zero<KY>();
        if constexpr (KX == kQ8) {
          xr[r][i] = on ? raw_load<KX>(a.q8.q, row * a.q8.ldq + c * 8) : raw_zero<KX>();
          eb[r][i] = on ? a.q8.e[row * a.q8.lde + (c >> 2)] : 0u;
        } else {
          xr[r][i] = on ? raw_load<KX>(a.x, row * a.ldx + c * 8) : raw_zero<KX>();
          eb[r][i] = 0u;
        }
        rr[r][i] = on && row < n_res ? raw_load<KD>(a.dres, row * a.lddr + c * 8) : raw_zero<KD>();
      }
    }
  };
  // The next rows are asked for as soon as these are in fp32 (wider rows have no registers
  // left for that): 1000003 x 128 from 8-bit rows with a residual, two rows at a time and three
  // CTAs an SM 171 us, so with one row and four CTAs 155
  constexpr bool kFetchAhead = NV == 1;
  const int64_t base0 = static_cast<int64_t>(blockIdx.x) * kTeams * R;
  if (kFetchAhead) fetch(base0);
  for (int64_t base = base0; base < n; base += step) {
    if (!kFetchAhead) fetch(base);
    float dy[R][NV][8], xh[R][NV][8], dot[R], rs[R];
    Raw8<KD> dr_raw[R][NV];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      dot[r] = 0.f;
      rs[r] = rs_next[r];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = i * TEAM + t;
        raw_values<KY>(yr[r][i], 0.f, dy[r][i]);
        raw_values<KX>(xr[r][i], group8_scale(eb[r][i]), xh[r][i]);
        dr_raw[r][i] = rr[r][i];
        mask8(dy[r][i], c, a.dim);
        mask8(xh[r][i], c, a.dim);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if constexpr (KX != kQ8) xh[r][i][j] *= rs[r];
          const float p = dy[r][i][j] * xh[r][i][j];
          acc[i][j] += p;
          dot[r] = fmaf(p, gam[i][j], dot[r]);
        }
      }
    }
    if (kFetchAhead && base + step < n) fetch(base + step);
    team_sum<TEAM, R>(dot, sh);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = base + r * kTeams + team;
      const float mean = dot[r] * inv_dim;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = i * TEAM + t;
        if (row < n && c < chunks) {
          float dr[8], o[8];
          raw_values<KD>(dr_raw[r][i], 0.f, dr);
#pragma unroll
          for (int j = 0; j < 8; ++j)
            o[j] = fmaf(rs[r], fmaf(-xh[r][i][j], mean, gam[i][j] * dy[r][i][j]), dr[j]);
          mask8(o, c, a.dim);
          if (a.clear_dy) {
            const float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            store_kind<KY>(a.dy, row * a.lddy + c * 8, z);
          }
          store_kind<KD>(a.dx, row * a.lddx + c * 8, o);
        }
      }
    }
  }
  // the CTA's column sums, its teams in order: into its part, or, when the grid is one
  // cluster, into shared memory, from which the cluster's CTAs finish them
  float* cols = parts + (kTeams > 1 ? kTeams * kCols : 0);
  float* out = a.cluster ? cols : a.work + static_cast<int64_t>(blockIdx.x) * a.dim;
  if constexpr (kTeams == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if ((i * TEAM + t) * 8 + j < a.dim) out[(i * TEAM + t) * 8 + j] = acc[i][j];
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) parts[team * kCols + (i * TEAM + t) * 8 + j] = acc[i][j];
    __syncthreads();
    for (int c = threadIdx.x; c < a.dim; c += kThreads) {
      float s = 0.f;
#pragma unroll 8
      for (int p = 0; p < kTeams; ++p) s += parts[p * kCols + c];
      out[c] = s;
    }
  }
  if (a.cluster) cluster_column_sums(cols, a.dim, a.dgamma, a.accumulate);
}

// one CTA per 32 columns; 32 threads a column, each a strided share of the parts
__global__ void __launch_bounds__(1024)
    sum_parts_kernel(const float* part, int parts, int64_t ld, int cols, float* out, bool accumulate) {
  GB_PDL_ENTRY();
  __shared__ float sh[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  if (c < cols) {
#pragma unroll 4
    for (int p = threadIdx.y; p < parts; p += 32) s += part[p * ld + c];
  }
  sh[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < cols) {
    float v = accumulate ? out[c] : 0.f;
    float w = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) w += sh[i][threadIdx.x];
    out[c] = v + w;
  }
}

// CTAs for cap rows: one pass of rows each, up to as many as the SMs hold at once.  Few rows
// are left to one cluster of up to eight CTAs, which joins its column sums over distributed
// shared memory: no second kernel, no work area (4.8 against 8.1 us a call for 64 x 64 rows).
constexpr int kBwdPasses = 2 * kClusterPasses;  // a pass is one row a team, half of what others take
template <int TEAM, int R>
int64_t passes(int cap) { return std::max<int64_t>(1, ceil_div(cap, kThreads / TEAM * R)); }

template <int K, int TEAM, int NV, int R>
void fwd_t(const RmsNormArgs& a, int num_sms, cudaStream_t stream) {
  const int64_t grid = std::min<int64_t>(passes<TEAM, R>(a.cap), static_cast<int64_t>(num_sms) * 4);
  launch_k(rmsnorm_fwd_kernel<K, TEAM, NV, R>, dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, stream, a);
  GB_LAUNCH_CHECK();
}

template <int K>
void fwd_k(const RmsNormArgs& a, int num_sms, cudaStream_t stream) {
  const int d = a.dim;
  if (d <= 32) return fwd_t<K, 4, 1, 2>(a, num_sms, stream);
  if (d <= 64) return fwd_t<K, 8, 1, 2>(a, num_sms, stream);
  if (d <= 128) return fwd_t<K, 16, 1, 2>(a, num_sms, stream);
  if (d <= 256) return fwd_t<K, 32, 1, 2>(a, num_sms, stream);
  if (d <= 512) return fwd_t<K, 64, 1, 2>(a, num_sms, stream);
  if (d <= 1024) return fwd_t<K, 128, 1, 2>(a, num_sms, stream);
  if (d <= 2048) return fwd_t<K, 256, 1, 2>(a, num_sms, stream);
  if (d <= 4096) return fwd_t<K, 256, 2, 1>(a, num_sms, stream);
  return fwd_t<K, 256, 4, 1>(a, num_sms, stream);
}

template <int KY, int KX, int KD, int TEAM, int NV, int R>
void bwd_t(RmsNormBwdArgs a, int num_sms, cudaStream_t stream) {
  const int64_t want = passes<TEAM, R>(a.cap);
  const size_t smem = sizeof(float) * ((TEAM < kThreads ? kThreads * NV * 8 : 0) + TEAM * NV * 8);
  auto kern = rmsnorm_bwd_kernel<KY, KX, KD, TEAM, NV, R>;
  if (want <= kBwdPasses) {
    a.cluster = true;
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(want, 8));
    launch_cluster_k(kern, dim3(grid), dim3(kThreads), grid, smem, stream, a);
    GB_LAUNCH_CHECK();
    return;
  }
  const int grid = static_cast<int>(std::min<int64_t>(want, static_cast<int64_t>(num_sms) * bwd_ctas(KY, KX, KD, NV)));
  launch_k(kern, dim3(grid), dim3(kThreads), smem, stream, a);
  GB_LAUNCH_CHECK();
  launch_sum_parts(a.work, grid, a.dim, a.dim, a.dgamma, a.accumulate, stream);
}

template <int KY, int KX, int KD>
void bwd_k(const RmsNormBwdArgs& a, int num_sms, cudaStream_t stream) {
  const int d = a.dim;
  if (d <= 64) return bwd_t<KY, KX, KD, 8, 1, 1>(a, num_sms, stream);
  if (d <= 128) return bwd_t<KY, KX, KD, 16, 1, 1>(a, num_sms, stream);
  if (d <= 256) return bwd_t<KY, KX, KD, 32, 1, 1>(a, num_sms, stream);
  if (d <= 512) return bwd_t<KY, KX, KD, 64, 1, 1>(a, num_sms, stream);
  if (d <= 1024) return bwd_t<KY, KX, KD, 128, 1, 1>(a, num_sms, stream);
  if (d <= 2048) return bwd_t<KY, KX, KD, 256, 1, 1>(a, num_sms, stream);
  if (d <= 4096) return bwd_t<KY, KX, KD, 256, 2, 1>(a, num_sms, stream);
  return bwd_t<KY, KX, KD, 256, 4, 1>(a, num_sms, stream);
}

template <int KY, int KX>
void bwd_yx(const RmsNormBwdArgs& a, int num_sms, cudaStream_t stream) {
  a.dx_f32 ? bwd_k<KY, KX, kF32>(a, num_sms, stream) : bwd_k<KY, KX, kBf>(a, num_sms, stream);
}
template <int KY>
void bwd_y(const RmsNormBwdArgs& a, int num_sms, cudaStream_t stream) {
  if (!a.x) return bwd_yx<KY, kQ8>(a, num_sms, stream);
  a.x_f32 ? bwd_yx<KY, kF32>(a, num_sms, stream) : bwd_yx<KY, kBf>(a, num_sms, stream);
}

}  // namespace

void launch_sum_parts(const float* part, int parts, int64_t ld, int cols, float* out, bool accumulate,
                      cudaStream_t stream) {
  launch_k(sum_parts_kernel, dim3(static_cast<unsigned>(ceil_div(cols, 32))), dim3(32, 32), 0, stream, part, parts, ld,
           cols, out, accumulate);
  GB_LAUNCH_CHECK();
}

int64_t rmsnorm_bwd_work_floats(int dim, int cap, int num_sms) {
  // rows of a CTA's pass, as bwd_k takes them
  const int rows = dim <= 64 ? 32 : dim <= 128 ? 16 : dim <= 256 ? 8 : dim <= 512 ? 4 : dim <= 1024 ? 2 : 1;
  const int64_t want = ceil_div(std::max(cap, 1), rows);
  return want <= kBwdPasses ? 0 : dim * std::min<int64_t>(want, static_cast<int64_t>(num_sms) * bwd_ctas(kBf, kBf, kBf, 1));
}

void launch_rmsnorm_fwd(const RmsNormArgs& a, int num_sms, cudaStream_t stream) {
  if (a.cap <= 0) return;
  a.f32 ? fwd_k<kF32>(a, num_sms, stream) : fwd_k<kBf>(a, num_sms, stream);
}

void launch_rmsnorm_bwd(const RmsNormBwdArgs& a, int num_sms, cudaStream_t stream) {
  a.dy_f32 ? bwd_y<kF32>(a, num_sms, stream) : bwd_y<kBf>(a, num_sms, stream);
}

}  // namespace dev
}  // namespace grappa
