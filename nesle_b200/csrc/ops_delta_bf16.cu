// ops_delta_bf16.cu -- the gated delta rule's kernels for one input type.
#include "ops_delta.cuh"

namespace nesle {
namespace ops {
namespace delta {
template int launch_forward<__nv_bfloat16>(const Scan&, cudaStream_t);
template int launch_backward<__nv_bfloat16>(const Scan&, cudaStream_t);
}  // namespace delta
}  // namespace ops
}  // namespace nesle
