// Which attention kernel a call takes.
#include "wlq_attn.cuh"
#include "wlq_internal.h"

namespace wlq {

namespace {
// A sequence's new rows of one kv head fill one or two MMA column blocks of
// the step kernel, or take the tensor-core tiles.  With 7, 8, 14 and 16 rows the
// step kernel is ahead by a tenth to a half (us, tiles' in brackets; 28 heads
// over 4, D 128; 7 rows: 32 sequences of 1280 in 8 bits 25 (42), in 16 bits 34
// (40), of 8192 73 (157) and 118 (132), one of 1500 16 (28); 14 rows: 32 (44), 37
// (40), 92 (159), 117 (132), 24 (29)) but for 14 rows over a single long sequence
// (16384 tokens in 16 bits: 38 (32), in 8 bits 37 (36)).
constexpr int kFewRows = 16;
bool few_rows(int64_t max_q, int G) { return max_q * G <= kFewRows; }
}  // namespace

size_t attention_workspace_bytes(int Hq, int Hkv, int D, int max_q) {
    const size_t sms = device_sm_count();
    // two parts per CTA of the step kernel (three CTAs per SM with 8 rows, two with 16), four CTAs' parts per SM of the tile
    // kernel
    const size_t rows = few_rows(max_q, Hq / Hkv) ? 2 * 2 * sms * kFewRows : 4 * sms * 256;
    return WLQ_ATTENTION_ZERO_BYTES + 64 * 1024 /* the tile kernel's list of joins */ + rows * (D + 4) * sizeof(float);
}

int launch_attention(const AttnParams& p, bool f16, cudaStream_t stream) {
    if (p.k_cache && few_rows(p.max_q, p.G))
        return f16 ? launch_attn_step_f16(p, stream) : launch_attn_step_bf16(p, stream);
    return f16 ? launch_attn_tile_f16(p, stream) : launch_attn_tile_bf16(p, stream);
}

// The attention kernels' device error words on the current device.
int attention_error(unsigned int* flags, int clear) {
    int (*const words[])(unsigned int*, int) = {attn_tile_error_f16, attn_tile_error_bf16, attn_step_error_f16,
                                                attn_step_error_bf16};
    unsigned int all = 0;
    for (auto word : words) {
        unsigned int v = 0;
        const int rc = word(&v, clear);
        if (rc) return rc;
        all |= v;
    }
    *flags = all;
    return WLQ_OK;
}

}  // namespace wlq
