// The linear layer's kernels with 128-column tiles (linear.cuh).
#include "linear.cuh"

namespace grappa {
namespace dev {

void launch_linear_128(const LinearArgs& a, cudaStream_t stream) { linear_tiles<128, 1>(a, stream); }

}  // namespace dev
}  // namespace grappa
