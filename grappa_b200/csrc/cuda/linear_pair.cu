// The linear layer's kernels with 256-column tiles of CTA pairs (linear.cuh).
#include "linear.cuh"

namespace grappa {
namespace dev {

void launch_linear_pair(const LinearArgs& a, cudaStream_t stream) { linear_tiles<256, 2>(a, stream); }

}  // namespace dev
}  // namespace grappa
