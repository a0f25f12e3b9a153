// group_norm_bwd_f32.cu - the backward group-norm kernels for float.
#include "group_norm_launch.cuh"

namespace bsx {
namespace norm {
template cudaError_t launch_bwd<float>(const Call&);
}  // namespace norm
}  // namespace bsx
