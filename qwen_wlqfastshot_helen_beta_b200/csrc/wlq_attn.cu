// Attention of packed prompts and of new tokens over a paged cache: a warp
// per (token, head), keys one after another with the running maximum and sum
// of a softmax in 32 bits.
#include <cfloat>

#include "wlq_attn.cuh"
#include "wlq_internal.h"

namespace wlq {

namespace {

template <typename T, int D, bool PAGED, bool QUANT>
__global__ void __launch_bounds__(128) attn_row_kernel(const AttnParams p) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int64_t tok = w / p.Hq;
    const int h = (int)(w - tok * p.Hq), hk = h / p.G;
    if (tok >= p.T) return;
    int b = (int)tok;
    int64_t first = tok, n = 1;
    if (p.cu) {
        int lo = 0, hi = p.B;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (p.cu[mid] <= tok) lo = mid;
            else hi = mid;
        }
        b = lo;
        first = p.cu[b];
        n = p.cu[b + 1] - first;
        if (tok < first || tok >= first + n) return;
    }
    int64_t len = n;
    if constexpr (PAGED) len = min((int64_t)p.kv_lens[b], p.table_cols * p.page_size);
    const int64_t seen = p.causal ? min(len, len - n + (tok - first) + 1) : len;
    float q[E], o[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        q[i] = ActTraits<T>::bits_to_f32(p.q[tok * p.q_tok + h * p.q_head + lane * E + i]) * p.scale_log2;
        o[i] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int64_t j = 0; j < seen; ++j) {
        float k[E], v[E];
        if constexpr (PAGED) {
            const int page = p.table[b * p.table_cols + (j >> p.log2_page)];
            const bool ok = page >= 0 && page < p.num_pages;
            const int64_t row = ((int64_t)page * p.Hkv + hk) * p.page_size + (j & (p.page_size - 1));
#pragma unroll
            for (int i = 0; i < E; ++i) {
                if constexpr (QUANT) {
                    float f[4], g[4];
                    e4m3x4_to_f32(ok ? reinterpret_cast<const uint8_t*>(p.k_cache)[row * D + lane * E + i] : 0, f);
                    e4m3x4_to_f32(ok ? reinterpret_cast<const uint8_t*>(p.v_cache)[row * D + lane * E + i] : 0, g);
                    k[i] = f[0] * exp2_biased(ok ? p.k_exp[row] : 127);
                    v[i] = g[0] * exp2_biased(ok ? p.v_exp[row] : 127);
                } else {
                    k[i] = ok ? ActTraits<T>::bits_to_f32(reinterpret_cast<const uint16_t*>(p.k_cache)[row * D + lane * E + i]) : 0.f;
                    v[i] = ok ? ActTraits<T>::bits_to_f32(reinterpret_cast<const uint16_t*>(p.v_cache)[row * D + lane * E + i]) : 0.f;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i) {
                k[i] = ActTraits<T>::bits_to_f32(p.k[(first + j) * p.k_tok + hk * p.k_head + lane * E + i]);
                v[i] = ActTraits<T>::bits_to_f32(p.v[(first + j) * p.v_tok + hk * p.v_head + lane * E + i]);
            }
        }
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) s += q[i] * k[i];
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        const float mn = fmaxf(m, s);
        const float c = exp2f(m - mn), e = exp2f(s - mn);
        l = l * c + e;
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] = o[i] * c + e * v[i];
        m = mn;
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const T r = ActTraits<T>::from_f32(seen > 0 ? o[i] * inv : 0.f);
        p.out[tok * p.o_tok + h * p.o_head + lane * E + i] = *reinterpret_cast<const uint16_t*>(&r);
    }
}

template <typename T, int D>
int run(const AttnParams& p, cudaStream_t s) {
    const unsigned grid = (unsigned)((p.T * p.Hq + 3) / 4);
    if (p.k_exp)
        attn_row_kernel<T, D, true, true><<<grid, 128, 0, s>>>(p);
    else
        attn_row_kernel<T, D, true, false><<<grid, 128, 0, s>>>(p);
    return check_cuda(cudaGetLastError(), "attn_row_kernel");
}

}  // namespace

namespace {
// A sequence's new rows of one kv head fill one MMA column block of the
// single-token kernel, or take the tensor-core tiles.
constexpr int kFewRows = 16;
bool few_rows(int64_t max_q, int G) { return max_q * G <= kFewRows; }
}  // namespace

size_t attention_workspace_bytes(int64_t T, int B, int Hq, int Hkv, int D, int max_q) {
    (void)T, (void)B;
    if (few_rows(max_q, Hq / Hkv)) return 0;
    return (size_t)device_sm_count() * 256 * (D + 2) * sizeof(float);
}

int launch_attention(const AttnParams& p, bool f16, cudaStream_t stream) {
    if (!p.k_cache || !few_rows(p.max_q, p.G)) return f16 ? launch_attn_tile_f16(p, stream) : launch_attn_tile_bf16(p, stream);
    if (f16) return p.D == 64 ? run<__half, 64>(p, stream) : run<__half, 128>(p, stream);
    return p.D == 64 ? run<__nv_bfloat16, 64>(p, stream) : run<__nv_bfloat16, 128>(p, stream);
}

}  // namespace wlq
