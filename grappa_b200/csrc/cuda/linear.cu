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
  // 8-bit z in brackets): 139058 x 128 x 256 20.4 / 21.1 [43.6 / 41.3], 139058 x 208 x 256
  // 26.4 / 32.8 [47.9 / 50.8], 139058 x 512 x 256 39 / 53 [59 / 66], 131072 x 1024 x 1024
  // 195 / 303 [258 / 354]; few tiles 20853 x 512 x 256 14.5 / 14.6 [22.6 / 20.7], 40000 x 208 x
  // 256 15.3 / 16.0 [29.1 / 26.2], 30000 x 512 x 256 15.1 / 18.1 [26.4 / 25.2], 20853 x 1024 x
  // 256 19.3 / 25.0 [26.3 / 28.8]; a third of the columns too many 139058 x 256 x 320
  // 44 / 41 [90 / 67], 139058 x 512 x 520 88 / 109 [143 / 144].
  const int64_t pairs = ceil_div(a.cap, 256) * ceil_div(a.N, 256);
  if (a.N > 128 && a.K >= 192 && pairs * a.K >= 384ll * sm_count() &&
      (a.K >= 512 || 2 * ceil_div(a.N, 256) == ceil_div(a.N, 128)))
    return launch_linear_pair(a, stream);
  // 128 / 64 columns: 300000 x 128 x 128 29 / 32 [56 / 64], 10240 x 512 x 256 9.2 / 9.3
  // [12.6 / 12.3], 3250 x 512 x 256 7.2 / 6.6 [9.8 / 8.7], N of 64 30 / 20 [56 / 36]
  if (a.N > 64 && ceil_div(a.cap, 128) * ceil_div(a.N, 128) >= sm_count()) return launch_linear_128(a, stream);
  return launch_linear_64(a, stream);
}

}  // namespace dev
}  // namespace grappa
