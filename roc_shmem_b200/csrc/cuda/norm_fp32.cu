// norm_fp32.cu — the norms' kernels for rows of type float (see norm_kernels.cuh).
#include "norm_kernels.cuh"

namespace bshmem {
namespace norms {
template int forward<float>(int, bool, const Params&, cudaStream_t);
template int backward<float>(int, bool, const Shape&, const BwdParams&, cudaStream_t);
}  // namespace norms
}  // namespace bshmem
