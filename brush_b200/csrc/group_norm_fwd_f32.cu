// group_norm_fwd_f32.cu - the forward group-norm kernels for float.
#include "group_norm_launch.cuh"

namespace bsx {
namespace norm {
template cudaError_t launch_fwd<float>(const Call&);
}  // namespace norm
}  // namespace bsx
