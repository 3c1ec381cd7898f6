// Backward pass of layer norm for float X, in a translation unit of its own (it builds beside the others).
#include "norm_grad.cuh"

namespace tca {
tcaspmm_status norm_backward_f32(const NormGradParams &p, int dim, long long *parts, cudaStream_t st)
{
    return norm_backward<float>(p, dim, parts, st);
}
}  // namespace tca
