// group_norm_f16.cu - the group-norm kernels for __half.
#include "group_norm_launch.cuh"

namespace bsx {
namespace norm {
template cudaError_t launch<__half>(const Call&);
}  // namespace norm
}  // namespace bsx
