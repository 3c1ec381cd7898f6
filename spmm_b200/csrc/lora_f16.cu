// Adapters of type __half, in a translation unit of its own (it builds beside the others).
#include "lora.cuh"

namespace tca {

tcaspmm_status lora_forward_f16(const ApplyParams &p, bool tokens, int sms, cudaStream_t st)
{
    return tokens ? token<__half>(p, st) : apply<__half, __half, false>(p, sms, st);
}

tcaspmm_status lora_input_grad_f16(const ApplyParams &p, bool in32, int sms, cudaStream_t st)
{
    return in32 ? apply<__half, float, true>(p, sms, st) : apply<__half, __half, true>(p, sms, st);
}

tcaspmm_status lora_factor_grads_f16(const GradParams &w, bool early, int sms, cudaStream_t st)
{
    return grads<__half>(w, early, sms, st);
}

}  // namespace tca
