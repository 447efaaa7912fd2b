// norm_fp16.cu — the norms' kernels for rows of type __half (see norm_kernels.cuh).
#include "norm_kernels.cuh"

namespace bshmem {
namespace norms {
template int forward<__half>(int, bool, const Params&, cudaStream_t);
template int backward<__half>(int, bool, const Shape&, const BwdParams&, cudaStream_t);
}  // namespace norms
}  // namespace bshmem
