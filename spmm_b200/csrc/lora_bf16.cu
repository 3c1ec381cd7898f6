// Adapters of type __nv_bfloat16, in a translation unit of its own (it builds beside the others).
#include "lora.cuh"

namespace tca {

tcaspmm_status lora_forward_bf16(const ApplyParams &p, bool tokens, int sms, cudaStream_t st)
{
    return tokens ? token<__nv_bfloat16>(p, st) : apply<__nv_bfloat16, __nv_bfloat16, false>(p, sms, st);
}

tcaspmm_status lora_input_grad_bf16(const ApplyParams &p, bool in32, int sms, cudaStream_t st)
{
    return in32 ? apply<__nv_bfloat16, float, true>(p, sms, st) : apply<__nv_bfloat16, __nv_bfloat16, true>(p, sms, st);
}

tcaspmm_status lora_factor_grads_bf16(const GradParams &w, bool early, int sms, cudaStream_t st)
{
    return grads<__nv_bfloat16>(w, early, sms, st);
}

}  // namespace tca
