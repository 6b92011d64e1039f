// Arguments and small device helpers shared by the attention operators: the
// paged cache's write and read (wlq_kv_cache.cu) and attention itself.
#pragma once

#include <cuda_fp8.h>

#include <algorithm>

#include "wlq_common.cuh"

namespace wlq {

constexpr int kReadTokens = 64;  // most tokens of one kv_read CTA

struct RopeParams {
    const uint16_t *q, *k, *v;  // [T, heads, D]; strides in elements, D contiguous
    uint16_t *q_out, *k_out;    // k_out may be null
    int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, qo_tok, qo_head, ko_tok, ko_head;
    const int64_t* positions;   // [T]
    const int64_t* slots;       // [T] page * page_size + offset, negative: not cached
    const float* cos_sin;       // [table_rows, rot]: rot / 2 cosines, rot / 2 sines
    void *k_cache, *v_cache;
    uint8_t *k_exp, *v_exp;
    int64_t T, table_rows, num_pages;
    int Hq, Hkv, D, rot, page_size, interleaved;
    int lanes_per_row, parts;   // set by the launcher
};

struct KvReadParams {
    const void *k_cache, *v_cache;
    const uint8_t *k_exp, *v_exp;
    const int32_t* table;  // [B, table_cols]
    const int32_t* cu;     // [B + 1] packed output rows of each sequence
    uint16_t *k_out, *v_out;
    int64_t T, num_pages, table_cols;
    int B, Hkv, D, page_size;
    int tokens;            // set by the launcher, as are the divisions' factors
    uint32_t per_magic, chunk_magic;
};

// One attention call.  Rows of a sequence are its new tokens times the G
// query heads of a kv head, token-major: row r is token r / G, head r % G.
struct AttnParams {
    const uint16_t* q;       // [T, Hq, D], strides in elements
    const uint16_t *k, *v;   // packed [T, Hkv, D] (prompt form)
    const void *k_cache, *v_cache;  // [pages, Hkv, page_size, D] (paged form)
    const uint8_t *k_exp, *v_exp;   // 8-bit caches
    uint16_t* out;           // [T, Hq, D]
    int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head;
    const int32_t* cu;       // [B + 1] packed query rows (null: one token per sequence)
    const int32_t* kv_lens;  // [B] (paged form)
    const int32_t* table;    // [B, table_cols]
    int64_t T, num_pages, table_cols;
    int B, Hq, Hkv, G, D, page_size, log2_page, causal;
    int max_q;               // upper bound of a sequence's new tokens (paged form)
    float scale_log2;        // softmax scale * log2(e): scores are kept in powers of two
    void* ws;                // workspace of the split forms
    size_t ws_bytes;
};

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (ActTraits<T>::kIsF16) {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}

// Read-only loads that are used once.  Not volatile, and called without a
// condition (at a valid address, the value dropped where it is not wanted): a
// load inside a branch is waited for where the branch ends, and sixteen of
// them take sixteen round trips.
__device__ __forceinline__ uint4 ldg16(const void* p) {
    uint4 r;
    asm("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
}
// 32 bytes a thread: a whole sector per store, half the instructions per byte
struct alignas(32) Words8 {
    uint32_t w[8];
};
__device__ __forceinline__ Words8 ldg32(const void* p) {
    Words8 r;
    asm("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
        : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]), "=r"(r.w[7])
        : "l"(p));
    return r;
}
__device__ __forceinline__ void stg32(void* p, const Words8& r) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"l"(p), "r"(r.w[0]), "r"(r.w[1]), "r"(r.w[2]), "r"(r.w[3]), "r"(r.w[4]), "r"(r.w[5]), "r"(r.w[6]),
                 "r"(r.w[7])
                 : "memory");
}
__device__ __forceinline__ uint4 keep_if(bool c, uint4 v) {
    return make_uint4(c ? v.x : 0u, c ? v.y : 0u, c ? v.z : 0u, c ? v.w : 0u);
}

// 2^(e - 127), e in 1..254
__device__ __forceinline__ float exp2_biased(uint32_t e) { return __uint_as_float(e << 23); }

// two e4m3 codes (the low 16 bits) -> two fp16 values, exact
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t w) {
    uint32_t d;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"((uint16_t)w));
    return d;
}
__device__ __forceinline__ void e4m3x4_to_f32(uint32_t w, float* f) {
    const uint32_t lo = e4m3x2_to_f16x2(w & 0xffffu), hi = e4m3x2_to_f16x2(w >> 16);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
}

}  // namespace wlq
