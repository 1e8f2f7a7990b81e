// ops_delta_f16.cu -- the gated delta rule's kernels for one input type.
#include "ops_delta.cuh"

namespace nesle {
namespace ops {
namespace delta {
template int launch_forward<__half>(const Scan&, cudaStream_t);
template int launch_backward<__half>(const Scan&, cudaStream_t);
}  // namespace delta
}  // namespace ops
}  // namespace nesle
