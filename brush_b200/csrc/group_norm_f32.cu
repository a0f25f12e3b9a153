// group_norm_f32.cu - the group-norm kernels for float.
#include "group_norm_launch.cuh"

namespace bsx {
namespace norm {
template cudaError_t launch<float>(const Call&);
}  // namespace norm
}  // namespace bsx
