// Tensor-core attention of many rows, f16 instances (a translation unit per
// activation type: they compile side by side).
#include "wlq_attn_tile.cuh"

namespace wlq {

int launch_attn_tile_f16(const AttnParams& p, cudaStream_t stream) { return launch_tile_any<__half>(p, stream); }

int attn_tile_error_f16(unsigned int* flags, int clear) { return tu_device_error(flags, clear); }

}  // namespace wlq
