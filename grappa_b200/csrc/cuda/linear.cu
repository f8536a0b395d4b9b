// Tile shape of the linear layer (kernels: linear.cuh).
#include "kernels.h"
#include "tcgen05.cuh"

namespace grappa {
namespace dev {

void launch_linear_fwd(const LinearArgs& a, cudaStream_t stream) {
  if (a.cap <= 0) return;
  // The pair's 256-column tiles read the operands least; two 128-column CTAs an SM overlap
  // the epilogues better.  So the pair takes what has enough products (K, and K times the
  // tiles) in tiles that are full enough.  Measured, pair / 128 columns, us (SiLU, residual and
  // 8-bit z in brackets): 139058 x 128 x 256 22.1 / 21.6 [45.7 / 42.8], 139058 x 208 x 256
  // 27.9 / 34.0 [49.5 / 51.4], 139058 x 512 x 256 43 / 54 [61 / 68], 131072 x 1024 x 1024
  // 216 / 309 [268 / 362]; few tiles 20853 x 512 x 256 14.8 / 14.1 [22.8 / 20.8], 40000 x 208 x
  // 256 12.4 / 13.2 [25.3 / 22.3], 30000 x 512 x 256 14.7 / 16.4 [24.1 / 24.1], 20853 x 1024 x
  // 256 22.4 / 26.8 [28.1 / 30.9]; a third of the columns too many 139058 x 256 x 320
  // 44 / 41 [94 / 68], 139058 x 512 x 520 97 / 111 [145 / 145].
  const int64_t pairs = ceil_div(a.cap, 256) * ceil_div(a.N, 256);
  if (a.N > 128 && a.K >= 192 && pairs * a.K >= 384ll * sm_count() &&
      (a.K >= 512 || 2 * ceil_div(a.N, 256) == ceil_div(a.N, 128)))
    return launch_linear_pair(a, stream);
  // 128 / 64 columns: 300000 x 128 x 128 30 / 33 [61 / 76], 10240 x 512 x 256 9.6 / 10.0
  // [13.3 / 13.9], N of 64 32 / 21 [62 / 45]
  if (a.N > 64 && ceil_div(a.cap, 128) * ceil_div(a.N, 128) >= sm_count()) return launch_linear_128(a, stream);
  return launch_linear_64(a, stream);
}

}  // namespace dev
}  // namespace grappa
