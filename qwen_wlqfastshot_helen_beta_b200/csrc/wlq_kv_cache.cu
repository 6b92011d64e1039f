// The paged k/v cache of an attention layer: rotary positions with the
// cache write (rope_kv_write_kernel) and the read-back (kv_read_kernel).
//
// Cache layout: [pages, kv_heads, page_size, D], one head's tokens of a page
// contiguous, so that an attention kernel fetches a page of one head as one
// 2-D tile.  16-bit caches hold the activation type.  8-bit caches hold e4m3
// codes and one byte e + 127 per row of D codes, e the smallest integer with
// max|x| <= 448 * 2^e.  The scale is a power of two on purpose: code * 2^e is
// a bf16 number (and an fp16 one in fp16's range), so whoever reads the cache
// dequantises into tensor-core operands without rounding a second time, and a
// floating format loses nothing to the coarse scale (its relative step does
// not depend on it).
//
// Both kernels are HBM-bound: every value is read once and written once.
// Measured, 28 heads over 4, D 128, 8-bit cache: the write of 32 prompts of 1024
// tokens (571 MB) 106 us, 5.4 TB/s, 82 % of the measured copy rate, one step of
// 32 tokens 3.0 us in a graph; the read-back of 180554 tokens (556 MB) 90 us, 6.2 TB/s, 94 %.
#include <cuda_fp8.h>

#include "wlq_attn.cuh"
#include "wlq_common.cuh"
#include "wlq_internal.h"

namespace wlq {

namespace {

constexpr int kRopeThreads = 128;
constexpr int kReadThreads = 256;

// Set when a token's position lies outside the cos/sin table; the token's
// outputs are then left as they were.
static __device__ unsigned int g_position_error = 0;

template <typename T>
__device__ __forceinline__ void unpack8(const uint4 w, float (&f)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = ActTraits<T>::bits_to_f32((uint16_t)u[i]);
        f[2 * i + 1] = ActTraits<T>::bits_to_f32((uint16_t)(u[i] >> 16));
    }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    return make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
}

// 16 bytes that this kernel may write later (q_out may be q): not by the read-only path
__device__ __forceinline__ uint4 ld16(const void* p) {
    uint4 r;
    asm("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
}

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}

// A warp takes one token (its cos/sin values stay in registers) and walks
// part of the token's heads, 32 / G rows at a time, kAhead such steps' loads in
// flight, then the next token: G lanes share a row, each with two 8-value chunks that hold both
// members of its pairs.  Few tokens spread their heads over several warps
// (`parts`), so that a decoding step is one round of loads.
constexpr int kAhead = 3;
constexpr int kRopeCtas = 4;  // per SM (at most 128 registers a thread)

template <typename T, bool QUANT, bool INTER>
__global__ void __launch_bounds__(kRopeThreads, kRopeCtas) rope_kv_write_kernel(const RopeParams p) {
    const int lane = threadIdx.x & 31;
    const int64_t w0 = (int64_t)blockIdx.x * (kRopeThreads / 32) + (threadIdx.x >> 5);
    const int64_t step = (int64_t)gridDim.x * (kRopeThreads / 32) / p.parts;  // tokens of a round
    const int part = (int)(w0 % p.parts);
    int64_t tok = w0 / p.parts;
    if (tok >= p.T) return;
    int64_t next_pos = p.positions[tok], next_slot = p.slots[tok];
    const int G = p.lanes_per_row, rows = 32 / G;
    const int l = lane & (G - 1), sub = lane / G;
    const bool live = 16 * l < p.D;  // D / 16 lanes work where G is rounded up
    const int nrot = p.rot >> 3;     // chunks that are rotated
    int ca, cb;                      // this lane's chunks
    if (INTER) {
        ca = l;
        cb = l + (p.D >> 4);
    } else if (l < nrot / 2) {
        ca = l;
        cb = l + nrot / 2;
    } else {
        ca = nrot + 2 * (l - nrot / 2);
        cb = ca + 1;
    }
    if (!live) ca = cb = 0;
    const int heads = p.Hq + 2 * p.Hkv;
    const int stride = p.parts * rows;
    uint4 xa[kAhead], xb[kAhead];
    auto load = [&](int h0) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int h = min(h0 + u * stride + sub, heads - 1);
            const uint16_t* src = h < p.Hq           ? p.q + tok * p.q_tok + h * p.q_head
                                  : h < p.Hq + p.Hkv ? p.k + tok * p.k_tok + (h - p.Hq) * p.k_head
                                                     : p.v + tok * p.v_tok + (h - p.Hq - p.Hkv) * p.v_head;
            xa[u] = ld16(src + 8 * ca);
            xb[u] = ld16(src + 8 * cb);
        }
    };
    for (; tok < p.T; tok += step) {
        load(part * rows);
        const int64_t pos = next_pos, slot = next_slot;
        if (tok + step < p.T) {  // the next token's, while this one is worked on
            next_pos = p.positions[tok + step];
            next_slot = p.slots[tok + step];
        }
        if (pos < 0 || pos >= p.table_rows) {
            if (lane == 0) atomicOr(&g_position_error, 1u);
            continue;
        }
        const bool store = slot >= 0 && slot < p.num_pages * p.page_size;  // a negative slot: a padding token
        const int64_t page = store ? slot / p.page_size : 0;
        const int off = store ? (int)(slot - page * p.page_size) : 0;

        // interleaved: 4 pairs of each chunk; halves: 8 pairs across the chunks
        float cs[8], sn[8];
        const float* row = p.cos_sin + pos * p.rot;
        const bool turn_a = live && ca < nrot, turn_b = live && cb < nrot;
#pragma unroll
        for (int i = 0; i < 8; ++i) cs[i] = 1.f, sn[i] = 0.f;
        {
            const int ia = INTER ? 4 * ca : 8 * ca, ib = INTER ? 4 * cb : 8 * ca + 4;
            if (turn_a) {
                const float4 c = *reinterpret_cast<const float4*>(row + ia);
                const float4 s = *reinterpret_cast<const float4*>(row + p.rot / 2 + ia);
                cs[0] = c.x, cs[1] = c.y, cs[2] = c.z, cs[3] = c.w;
                sn[0] = s.x, sn[1] = s.y, sn[2] = s.z, sn[3] = s.w;
            }
            if (turn_b) {
                const float4 c = *reinterpret_cast<const float4*>(row + ib);
                const float4 s = *reinterpret_cast<const float4*>(row + p.rot / 2 + ib);
                cs[4] = c.x, cs[5] = c.y, cs[6] = c.z, cs[7] = c.w;
                sn[4] = s.x, sn[5] = s.y, sn[6] = s.z, sn[7] = s.w;
            }
        }

        for (int h0 = part * rows; h0 < heads; h0 += kAhead * stride) {
            if (h0 != part * rows) load(h0);
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                if (h0 + u * stride >= heads) break;  // uniform over the warp
                const int h = h0 + u * stride + sub;
                const bool ok = live && h < heads;
                const int kind = h < p.Hq ? 0 : (h < p.Hq + p.Hkv ? 1 : 2);  // q, k, v
                const int hh = kind == 0 ? h : (kind == 1 ? h - p.Hq : h - p.Hq - p.Hkv);
                float a[8], b[8];
                unpack8<T>(keep_if(ok, xa[u]), a);
                unpack8<T>(keep_if(ok, xb[u]), b);
                if (kind != 2) {
                    if (INTER) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float x = a[2 * i], y = a[2 * i + 1], z = b[2 * i], t = b[2 * i + 1];
                            if (turn_a) {
                                a[2 * i] = x * cs[i] - y * sn[i];
                                a[2 * i + 1] = y * cs[i] + x * sn[i];
                            }
                            if (turn_b) {
                                b[2 * i] = z * cs[4 + i] - t * sn[4 + i];
                                b[2 * i + 1] = t * cs[4 + i] + z * sn[4 + i];
                            }
                        }
                    } else if (turn_a) {  // both chunks are rotated, or neither
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float x = a[i], y = b[i];
                            a[i] = x * cs[i] - y * sn[i];
                            b[i] = y * cs[i] + x * sn[i];
                        }
                    }
                }
                uint16_t* d = kind == 0   ? p.q_out + tok * p.qo_tok + hh * p.qo_head
                              : kind == 1 ? p.k_out + tok * p.ko_tok + hh * p.ko_head
                                          : nullptr;
                if (ok && (kind == 0 || (kind == 1 && p.k_out))) {
                    *reinterpret_cast<uint4*>(d + 8 * ca) = pack8<T>(a);
                    *reinterpret_cast<uint4*>(d + 8 * cb) = pack8<T>(b);
                }
                if (!store || h0 + u * stride + rows <= p.Hq) continue;  // uniform over the warp
                const int64_t crow = (page * p.Hkv + hh) * p.page_size + off;
                if constexpr (QUANT) {
                    if (ActTraits<T>::kIsF16) {
                        // the largest e4m3 grid value below 65504, so that what is read back stays finite in fp16
                        // (a NaN passes, and becomes the NaN code)
                        auto within = [](float x) { return fabsf(x) > 61440.f ? copysignf(61440.f, x) : x; };
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            a[i] = within(a[i]);
                            b[i] = within(b[i]);
                        }
                    }
                    float top = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) top = fmaxf(top, fmaxf(fabsf(a[i]), fabsf(b[i])));
                    for (int x = 1; x < G; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                    // top = m 2^x with m in [1, 2) and 448 = 1.75 * 2^8
                    const uint32_t bits = __float_as_uint(top);
                    const int e = max(1, (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0));  // + 127
                    const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
                    if (ok && kind != 0) {
                        uint8_t* c8 = reinterpret_cast<uint8_t*>(kind == 1 ? p.k_cache : p.v_cache) + crow * p.D;
                        *reinterpret_cast<uint2*>(c8 + 8 * ca) =
                            make_uint2(e4m3x4(a[0] * inv, a[1] * inv, a[2] * inv, a[3] * inv),
                                       e4m3x4(a[4] * inv, a[5] * inv, a[6] * inv, a[7] * inv));
                        *reinterpret_cast<uint2*>(c8 + 8 * cb) =
                            make_uint2(e4m3x4(b[0] * inv, b[1] * inv, b[2] * inv, b[3] * inv),
                                       e4m3x4(b[4] * inv, b[5] * inv, b[6] * inv, b[7] * inv));
                        if (l == 0) (kind == 1 ? p.k_exp : p.v_exp)[crow] = (uint8_t)e;
                    }
                } else if (ok && kind != 0) {
                    uint16_t* c16 = reinterpret_cast<uint16_t*>(kind == 1 ? p.k_cache : p.v_cache) + crow * p.D;
                    *reinterpret_cast<uint4*>(c16 + 8 * ca) = pack8<T>(a);
                    *reinterpret_cast<uint4*>(c16 + 8 * cb) = pack8<T>(b);
                }
            }
        }
    }
}

// A CTA reads back `tokens` consecutive rows of the packed output, all heads
// of k or of v: the first threads look the rows' cache slots up, then every
// thread moves 16 values per item (16 codes or 32 bytes in, one 32-byte store
// out), four items' loads in flight.  Rows outside the table or the pool are
// zeros.
//
// WIDE: outputs, and caches of 16 bits, that begin at a multiple of 32 bytes
// (items are 32 bytes, so all of them then do).  The others, which need only
// be 16-byte aligned, are moved as two halves: 115 us against 92 for 180000
// tokens of an 8-bit cache, 138 against 119 from a 16-bit one, cold L2.
template <typename T, bool QUANT, bool WIDE>
__global__ void __launch_bounds__(kReadThreads) kv_read_kernel(const KvReadParams p) {
    __shared__ int64_t base[kReadTokens];  // cache row of head 0, or -1
    const int64_t t0 = (int64_t)blockIdx.x * p.tokens;
    const int nt = (int)min((int64_t)p.tokens, p.T - t0);
    if ((int)threadIdx.x < nt) {
        const int64_t t = t0 + threadIdx.x;
        int lo = 0, hi = p.B;  // last sequence with cu[lo] <= t
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (p.cu[mid] <= t) lo = mid;
            else hi = mid;
        }
        const int64_t pos = t - p.cu[lo];
        const int64_t pg = pos / p.page_size;
        int64_t r = -1;
        if (pos >= 0 && t < p.cu[lo + 1] && pg < p.table_cols) {
            const int id = p.table[(int64_t)lo * p.table_cols + pg];
            if (id >= 0 && id < p.num_pages) r = (int64_t)id * p.Hkv * p.page_size + (pos - pg * p.page_size);
        }
        base[threadIdx.x] = r;
    }
    __syncthreads();
    const int per = p.Hkv * (p.D >> 4);  // items of one token
    const int n = nt * per;
    constexpr int U = 4;
    const int which = blockIdx.y;  // k, v
    const uint8_t* src = reinterpret_cast<const uint8_t*>(which ? p.v_cache : p.k_cache);
    const uint8_t* exps = which ? p.v_exp : p.k_exp;
    uint16_t* dst = (which ? p.v_out : p.k_out) + t0 * per * 16;
    for (int i0 = threadIdx.x; i0 < n; i0 += U * kReadThreads) {
        Words8 w[U];
        uint32_t e[U];
        bool in[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = min(i0 + u * kReadThreads, n - 1);
            const int tk = p.per_magic ? __umulhi((uint32_t)i, p.per_magic) : i;
            const int x = i - tk * per;
            const int h = p.chunk_magic ? __umulhi((uint32_t)x, p.chunk_magic) : x;
            const int64_t r = base[tk];
            in[u] = r >= 0;
            const int64_t row = in[u] ? r + (int64_t)h * p.page_size : 0;
            const int64_t at = row * p.D + 16 * (x - h * (p.D >> 4));
            if constexpr (QUANT) {
                const uint4 q = ldg16(src + at);
                w[u].w[0] = q.x, w[u].w[1] = q.y, w[u].w[2] = q.z, w[u].w[3] = q.w;
                e[u] = __ldg(exps + row);
            } else if constexpr (WIDE) {
                w[u] = ldg32(src + at * 2);
            } else {
                const uint4 a = ldg16(src + at * 2), b = ldg16(src + at * 2 + 16);
                w[u] = Words8{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            Words8 o = w[u];
            if constexpr (QUANT) {
                const float s = exp2_biased(e[u]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float f[4];
                    e4m3x4_to_f32(w[u].w[j], f);
                    o.w[2 * j] = pack2<T>(f[0] * s, f[1] * s);
                    o.w[2 * j + 1] = pack2<T>(f[2] * s, f[3] * s);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) o.w[j] = in[u] ? o.w[j] : 0u;
            const int i = i0 + u * kReadThreads;
            uint16_t* d = dst + (int64_t)i * 16;
            if (i < n) {
                if constexpr (WIDE) {
                    stg32(d, o);
                } else {
                    *reinterpret_cast<uint4*>(d) = make_uint4(o.w[0], o.w[1], o.w[2], o.w[3]);
                    *reinterpret_cast<uint4*>(d + 8) = make_uint4(o.w[4], o.w[5], o.w[6], o.w[7]);
                }
            }
        }
    }
}

// q = i / d for i < n as a multiply-high, exact while n * d < 2^32; 0 stands for d = 1
uint32_t magic_u32(uint32_t d) { return d == 1 ? 0u : (uint32_t)((0x100000000ull + d - 1) / d); }

}  // namespace

int launch_rope_kv_write(RopeParams& p, bool f16, bool quant, cudaStream_t stream) {
    p.lanes_per_row = 1;
    while (p.lanes_per_row * 16 < p.D) p.lanes_per_row <<= 1;
    const int steps = (p.Hq + 2 * p.Hkv + 32 / p.lanes_per_row - 1) / (32 / p.lanes_per_row);
    // enough warps for 16 per SM before a warp walks several steps (28 heads over 4, D 128, 8-bit, in a graph: 1 to 32
    // tokens 2.7 us, 5.2 with a warp a token; 300 tokens 4.5 and 5.5; 4000 the same)
    const int64_t want = (int64_t)device_sm_count() * 16;
    const int64_t resident = (int64_t)device_sm_count() * kRopeCtas;
    p.parts = (int)std::min(std::min<int64_t>(steps, resident), std::max<int64_t>(1, (want + p.T - 1) / p.T));
    // CTAs that fit at once; their warps walk the tokens (a multiple of `parts` warps: the same part each time)
    const int64_t warps = p.T * p.parts, per = kRopeThreads / 32;
    const unsigned grid = (unsigned)std::min((warps + per - 1) / per, resident / p.parts * p.parts);
    auto run = [&](auto kernel) { kernel<<<grid, kRopeThreads, 0, stream>>>(p); };
    auto typed = [&](auto t) {
        using T = decltype(t);
        if (quant)
            p.interleaved ? run(rope_kv_write_kernel<T, true, true>) : run(rope_kv_write_kernel<T, true, false>);
        else
            p.interleaved ? run(rope_kv_write_kernel<T, false, true>) : run(rope_kv_write_kernel<T, false, false>);
    };
    f16 ? typed(__half{}) : typed(__nv_bfloat16{});
    return check_cuda(cudaGetLastError(), "rope_kv_write_kernel");
}

int launch_kv_read(KvReadParams& p, bool f16, bool quant, cudaStream_t stream) {
    // A CTA takes the tokens of one round of its threads (four items each); few rows, 8 tokens, which start more CTAs.  4
    // heads of 128, 8 bits, in a graph: 500 rows 2.7 us with 8 tokens and 2.8 with 32, 1500 rows 3.7 and 3.1, 16000 17.4 and
    // 7.8, 100000 104 and 50 (51 with 64); 8 heads 115 with 8, 96 with 16, 100 with 64; 2 heads of 64 41 with 8, 15 with 64.
    p.tokens = p.T < 1000 ? 8 : std::clamp(4 * kReadThreads / (p.Hkv * (p.D >> 4)), 8, kReadTokens);
    p.per_magic = magic_u32((uint32_t)(p.Hkv * (p.D >> 4)));
    p.chunk_magic = magic_u32((uint32_t)(p.D >> 4));
    const dim3 grid((unsigned)((p.T + p.tokens - 1) / p.tokens), 2);
    auto bits = [](const void* a) { return reinterpret_cast<uintptr_t>(a); };
    const bool wide = ((bits(p.k_out) | bits(p.v_out) | (quant ? 0 : bits(p.k_cache) | bits(p.v_cache))) & 31) == 0;
    auto run = [&](auto kernel) { kernel<<<grid, kReadThreads, 0, stream>>>(p); };
    auto typed = [&](auto t) {
        using T = decltype(t);
        if (quant)
            wide ? run(kv_read_kernel<T, true, true>) : run(kv_read_kernel<T, true, false>);
        else
            wide ? run(kv_read_kernel<T, false, true>) : run(kv_read_kernel<T, false, false>);
    };
    f16 ? typed(__half{}) : typed(__nv_bfloat16{});
    return check_cuda(cudaGetLastError(), "kv_read_kernel");
}

// Reads (and with `clear` zeroes) the position error of the current device.
int rope_position_error(unsigned int* flag, int clear) {
    unsigned int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, g_position_error, sizeof(v));
    if (e == cudaSuccess && clear && v) {
        const unsigned int z = 0;
        e = cudaMemcpyToSymbol(g_position_error, &z, sizeof(z));
    }
    if (e != cudaSuccess) return check_cuda(e, "position error word");
    *flag = v;
    return WLQ_OK;
}

}  // namespace wlq
