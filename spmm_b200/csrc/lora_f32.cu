// Adapters of type float, in a translation unit of its own (it builds beside the others).
#include "lora.cuh"

namespace tca {

tcaspmm_status lora_forward_f32(const ApplyParams &p, bool tokens, int sms, cudaStream_t st)
{
    return tokens ? token<float>(p, st) : apply<float, float, false>(p, sms, st);
}

tcaspmm_status lora_input_grad_f32(const ApplyParams &p, bool in32, int sms, cudaStream_t st)
{
    return in32 ? apply<float, float, true>(p, sms, st) : apply<float, float, true>(p, sms, st);
}

tcaspmm_status lora_factor_grads_f32(const GradParams &w, bool early, int sms, cudaStream_t st)
{
    return grads<float>(w, early, sms, st);
}

}  // namespace tca
