// Attention of few rows over the paged cache, bf16 instances.
#include "wlq_attn_step.cuh"

namespace wlq {

int launch_attn_step_bf16(const AttnParams& p, cudaStream_t stream) { return launch_step_any<__nv_bfloat16>(p, stream); }

int attn_step_error_bf16(unsigned int* flags, int clear) { return tu_device_error(flags, clear); }

}  // namespace wlq
