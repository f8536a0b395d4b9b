// The linear layer's kernels with 64-column tiles (linear.cuh).
#include "linear.cuh"

namespace grappa {
namespace dev {

void launch_linear_64(const LinearArgs& a, cudaStream_t stream) { linear_tiles<64, 1>(a, stream); }

}  // namespace dev
}  // namespace grappa
