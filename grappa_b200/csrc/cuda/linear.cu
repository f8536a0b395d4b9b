// Tile shape of the linear layer (kernels: linear.cuh).
#include "kernels.h"
#include "tcgen05.cuh"

namespace grappa {
namespace dev {

void launch_linear_fwd(const LinearArgs& a, cudaStream_t stream) {
  if (a.cap <= 0) return;
  // Long products (K from 384 on) want the pair's 256-column tiles, which read the operands
  // least; short ones are bound by their rows' way through HBM and the epilogue, and two
  // 128-column CTAs an SM overlap those better.  Measured, pair / 128 columns, us (SiLU,
  // residual and 8-bit z in brackets): 139058 x 208 x 256 37 / 35 [63 / 50], 139058 x 512 x 256
  // 46 / 52 [71 / 68], 65536 x 1024 x 512 64 / 78 [82 / 93], 131072 x 1024 x 1024 237 / 307
  // [303 / 360].  Fewer tiles than SMs: the narrowest (10240 x 512 x 256: 14 / 11, 64 columns 12).
  if (a.K >= 384 && a.N > 128 && ceil_div(a.cap, 256) * ceil_div(a.N, 256) >= sm_count() / 2)
    return launch_linear_pair(a, stream);
  if (a.N > 64 && ceil_div(a.cap, 128) * ceil_div(a.N, 128) >= sm_count()) return launch_linear_128(a, stream);
  return launch_linear_64(a, stream);
}

}  // namespace dev
}  // namespace grappa
