// group_norm_bwd_bf16.cu - the backward group-norm kernels for __nv_bfloat16.
#include "group_norm_launch.cuh"

namespace bsx {
namespace norm {
template cudaError_t launch_bwd<__nv_bfloat16>(const Call&);
}  // namespace norm
}  // namespace bsx
