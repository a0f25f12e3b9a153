// group_norm_fwd_f16.cu - the forward group-norm kernels for __half.
#include "group_norm_launch.cuh"

namespace bsx {
namespace norm {
template cudaError_t launch_fwd<__half>(const Call&);
}  // namespace norm
}  // namespace bsx
