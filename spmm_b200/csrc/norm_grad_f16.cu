// Backward pass of layer norm for __half X, in a translation unit of its own (it builds beside the others).
#include "norm_grad.cuh"

namespace tca {
tcaspmm_status norm_backward_f16(const NormGradParams &p, int dim, long long *parts, cudaStream_t st)
{
    return norm_backward<__half>(p, dim, parts, st);
}
}  // namespace tca
