// group_norm_bwd_f16.cu - the backward group-norm kernels for __half.
#include "group_norm_launch.cuh"

namespace bsx {
namespace norm {
template cudaError_t launch_bwd<__half>(const Call&);
}  // namespace norm
}  // namespace bsx
