// Pieces that both attention kernels use: waits, copies, exponentials, and a
// row computed by one warp alone.
#pragma once

#include "wlq_attn.cuh"
#include "wlq_once.h"
#include "wlq_sm100.cuh"

namespace wlq {

namespace {

// Where k and v lie: packed rows, a 16-bit paged cache, an 8-bit one.
enum KvSource { kPacked = 0, kPaged = 1, kPaged8 = 2 };

// mbar_wait by a whole warp, which goes on or gives up together.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

__device__ __forceinline__ uint32_t lds8(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
// Arrives on bar when this thread's cp.async copies so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ int64_t warp_sum(int64_t v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
__device__ __forceinline__ int warp_scan(int v, int lane) {  // inclusive
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += o;
    }
    return v;
}

// The sequence and kv head a row belongs to, the sequence's first row in q.
struct RowOf {
    int b, hk, first;
};

// Lane values of one cached or packed row in fp32 (E = D / 32 each).
template <typename T, int D, int SRC>
__device__ __forceinline__ void load_row(const AttnParams& p, const RowOf& u, int j, bool v, int lane,
                                         float (&f)[D / 32]) {
    constexpr int E = D / 32;
#pragma unroll
    for (int i = 0; i < E; ++i) f[i] = 0.f;
    if constexpr (SRC == kPacked) {
        const uint16_t* s = v ? p.v + (int64_t)(u.first + j) * p.v_tok + u.hk * p.v_head
                              : p.k + (int64_t)(u.first + j) * p.k_tok + u.hk * p.k_head;
#pragma unroll
        for (int i = 0; i < E; ++i) f[i] = ActTraits<T>::bits_to_f32(s[lane * E + i]);
    } else {
        const int page = p.table[(int64_t)u.b * p.table_cols + (j >> p.log2_page)];
        if (page < 0 || page >= p.num_pages) return;
        const int64_t row = ((int64_t)page * p.Hkv + u.hk) * p.page_size + (j & (p.page_size - 1));
        if constexpr (SRC == kPaged) {
            const uint16_t* s = static_cast<const uint16_t*>(v ? p.v_cache : p.k_cache) + row * D;
#pragma unroll
            for (int i = 0; i < E; ++i) f[i] = ActTraits<T>::bits_to_f32(s[lane * E + i]);
        } else {
            const uint8_t* s = static_cast<const uint8_t*>(v ? p.v_cache : p.k_cache) + row * D;
            const float e = exp2_biased((v ? p.v_exp : p.k_exp)[row]);
#pragma unroll
            for (int i = 0; i < E; ++i) {
                float g[4];
                e4m3x4_to_f32(s[lane * E + i], g);
                f[i] = g[0] * e;
            }
        }
    }
}

// The last of the keys [j0, j1) whose v, as the 16-bit values the tensor cores
// take, is not finite throughout; -1 if there is none.  By one warp, a key a lane.
template <typename T, int D, int SRC>
__device__ __noinline__ int last_not_finite(const AttnParams& p, const RowOf& u, int j0, int j1, int lane) {
    for (int hi = j1; hi > j0; hi -= 32) {
        const int j = hi - 1 - lane;
        bool bad = false;
        if (j >= j0) {
            int64_t row = 0;
            bool there = true;
            if constexpr (SRC != kPacked) {
                const int page = p.table[(int64_t)u.b * p.table_cols + (j >> p.log2_page)];
                there = page >= 0 && page < p.num_pages;  // a page outside the pool reads as zeros
                if (there) row = ((int64_t)page * p.Hkv + u.hk) * p.page_size + (j & (p.page_size - 1));
            }
            if constexpr (SRC == kPaged8) {
                const uint8_t* s = static_cast<const uint8_t*>(p.v_cache) + row * D;
                uint32_t top = 0;  // the largest code without its sign, a byte each
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    const uint4 w = ldg16(s + 16 * i);
                    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int y = 0; y < 4; ++y) top = __vmaxu4(top, x[y] & 0x7f7f7f7fu);
                }
                top = max(max(top & 0xff, (top >> 8) & 0xff), max((top >> 16) & 0xff, top >> 24));
                const uint32_t e = p.v_exp[row];
                float f[4];
                e4m3x4_to_f32(top, f);
                const uint32_t v = pack2<T>(f[0] * exp2_biased(e), 0.f);
                bad = e == 255 || !isfinite(ActTraits<T>::bits_to_f32((uint16_t)v));
            } else {
                const uint16_t* s = SRC == kPacked ? p.v + (int64_t)(u.first + j) * p.v_tok + u.hk * p.v_head
                                                   : static_cast<const uint16_t*>(p.v_cache) + row * D;
                uint32_t top = 0;  // the largest value without its sign, two bytes each
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    const uint4 w = ldg16(s + 8 * i);
                    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int y = 0; y < 4; ++y) top = __vmaxu2(top, x[y] & 0x7fff7fffu);
                }
                bad = max(top & 0xffffu, top >> 16) >= (ActTraits<T>::kIsF16 ? 0x7c00u : 0x7f80u);
            }
            bad = bad && there;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, bad);
        if (hit) return hi - __ffs(hit);
    }
    return -1;
}

// One row over its keys [j0, j1) without the tensor cores, by one warp.  A
// tensor-core product multiplies the values of keys a row does not see by
// zero; where those are infinite or NaN the product is NaN, and the row is
// computed here instead.  m is in powers of two.  It takes about 0.5 us a key,
// so the callers look for such a value first: a NaN that the rows do see is
// no reason (a prompt of 4096 tokens with one took 58 ms, 0.12 without).
template <typename T, int D, int SRC>
__device__ __noinline__ void row_alone(const AttnParams& p, const RowOf& u, int row, int j0, int j1, int lane,
                                       float (&o)[D / 32], float& m, float& l) {
    constexpr int E = D / 32;
    const int h = u.hk * p.G + row % p.G;
    const int64_t tok = u.first + row / p.G;
    float q[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        q[i] = ActTraits<T>::bits_to_f32(p.q[tok * p.q_tok + h * p.q_head + lane * E + i]);
        o[i] = 0.f;
    }
    m = -INFINITY;
    l = 0.f;
    for (int j = j0; j < j1; ++j) {
        float k[E], v[E];
        load_row<T, D, SRC>(p, u, j, false, lane, k);
        load_row<T, D, SRC>(p, u, j, true, lane, v);
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) s += q[i] * k[i];
#pragma unroll
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        s *= p.scale_log2;
        const float mn = fmaxf(m, s);
        const float ref = mn == -INFINITY ? 0.f : mn;
        const float c = exp2f(m - ref), e = exp2f(s - ref);
        l = l * c + e;
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] = o[i] * c + e * v[i];
        m = mn;
        // NaN everywhere: whatever follows, the row stays so
        bool nan = true;
#pragma unroll
        for (int i = 0; i < E; ++i) nan = nan && o[i] != o[i];
        if (__all_sync(0xffffffffu, nan)) return;
    }
}

// Raises a kernel's dynamic shared memory limit on the current device.
template <typename Kernel>
int allow_shared_memory(OncePerDevice& limit, Kernel kernel, int bytes, const char* what) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess)
        e = limit.run(device, [&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); });
    return check_cuda(e, what);
}

}  // namespace

}  // namespace wlq
