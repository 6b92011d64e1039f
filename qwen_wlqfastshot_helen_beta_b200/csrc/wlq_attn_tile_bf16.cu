// Tensor-core attention of many rows, bf16 instances (a translation unit per
// activation type: they compile side by side).
#include "wlq_attn_tile.cuh"

namespace wlq {

int launch_attn_tile_bf16(const AttnParams& p, cudaStream_t stream) { return launch_tile_any<__nv_bfloat16>(p, stream); }

int attn_tile_error_bf16(unsigned int* flags, int clear) { return tu_device_error(flags, clear); }

}  // namespace wlq
