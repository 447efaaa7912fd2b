// norm_bf16.cu — the norms' kernels for rows of type __nv_bfloat16 (see norm_kernels.cuh).
#include "norm_kernels.cuh"

namespace bshmem {
namespace norms {
template int forward<__nv_bfloat16>(int, bool, const Params&, cudaStream_t);
template int backward<__nv_bfloat16>(int, bool, const Shape&, const BwdParams&, cudaStream_t);
}  // namespace norms
}  // namespace bshmem
