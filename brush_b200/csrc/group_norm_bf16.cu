// group_norm_bf16.cu - the group-norm kernels for __nv_bfloat16.
#include "group_norm_launch.cuh"

namespace bsx {
namespace norm {
template cudaError_t launch<__nv_bfloat16>(const Call&);
}  // namespace norm
}  // namespace bsx
