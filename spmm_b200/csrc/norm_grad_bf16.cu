// Backward pass of layer norm for __nv_bfloat16 X, in a translation unit of its own (it builds beside the others).
#include "norm_grad.cuh"

namespace tca {
tcaspmm_status norm_backward_bf16(const NormGradParams &p, int dim, long long *parts, cudaStream_t st)
{
    return norm_backward<__nv_bfloat16>(p, dim, parts, st);
}
}  // namespace tca
