// group_norm_fwd_bf16.cu - the forward group-norm kernels for __nv_bfloat16.
#include "group_norm_launch.cuh"

namespace bsx {
namespace norm {
template cudaError_t launch_fwd<__nv_bfloat16>(const Call&);
}  // namespace norm
}  // namespace bsx
