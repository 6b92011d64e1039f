// extern "C" entry points of the attention operators: argument validation
// and dispatch.  No counterpart in the reference, which leaves what stands
// between the qkv and the o projection to vLLM.
#include <cmath>
#include <cstring>

#include "wlq_attn.cuh"
#include "wlq_internal.h"

namespace wlq {

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int bad_dtype(const char* fn, int dtype) {
    if (dtype == WLQ_DTYPE_F16 || dtype == WLQ_DTYPE_BF16) return WLQ_OK;
    return fail(WLQ_ERR_UNSUPPORTED, "%s: act_dtype must be WLQ_DTYPE_F16 or WLQ_DTYPE_BF16 (got %d)", fn, dtype);
}

// A [T, heads, D] tensor: 16-byte aligned rows.
int bad_rows(const char* fn, const char* what, const void* p, int64_t tok, int64_t head) {
    if (!p) return fail(WLQ_ERR_INVALID_ARG, "%s: %s is required", fn, what);
    if (!aligned16(p) || tok % 8 || head % 8)
        return fail(WLQ_ERR_ALIGNMENT,
                    "%s: the rows of %s must be 16-byte aligned (token stride %lld, head stride %lld elements)", fn,
                    what, (long long)tok, (long long)head);
    if (tok < 0 || head < 0)
        return fail(WLQ_ERR_INVALID_ARG, "%s: %s has a negative stride", fn, what);
    return WLQ_OK;
}

int bad_heads(const char* fn, int Hq, int Hkv) {
    if (Hq < 1 || Hkv < 1 || Hq > 65535 || Hq % Hkv)
        return fail(WLQ_ERR_INVALID_ARG, "%s: %d query heads over %d kv heads", fn, Hq, Hkv);
    return WLQ_OK;
}

int bad_cache(const char* fn, const void* k, const void* v, const void* ke, const void* ve, int64_t pages, int ps) {
    if (!k || !v) return fail(WLQ_ERR_INVALID_ARG, "%s: k_cache and v_cache are required", fn);
    if (!ke != !ve) return fail(WLQ_ERR_INVALID_ARG, "%s: give k_exp and v_exp (8-bit caches) or neither", fn);
    if (!aligned16(k) || !aligned16(v)) return fail(WLQ_ERR_ALIGNMENT, "%s: the caches must be 16-byte aligned", fn);
    if (ps != 16 && ps != 32 && ps != 64 && ps != 128)
        return fail(WLQ_ERR_UNSUPPORTED, "%s: page_size must be 16, 32, 64 or 128 (got %d)", fn, ps);
    if (pages < 1 || pages > 0x7fffffff) return fail(WLQ_ERR_INVALID_ARG, "%s: %lld pages", fn, (long long)pages);
    return WLQ_OK;
}

int log2_of(int v) {
    int n = 0;
    while ((1 << n) < v) ++n;
    return n;
}

}  // namespace

}  // namespace wlq

using namespace wlq;

extern "C" {

int wlq_rope_kv_write(const void* q, const void* k, const void* v, const int64_t* positions, const float* cos_sin,
                      const int64_t* slots, void* k_cache, void* v_cache, uint8_t* k_exp, uint8_t* v_exp, void* q_out,
                      void* k_out, int64_t q_tok, int64_t q_head, int64_t k_tok, int64_t k_head, int64_t v_tok,
                      int64_t v_head, int64_t qo_tok, int64_t qo_head, int64_t ko_tok, int64_t ko_head, int64_t T,
                      int64_t table_rows, int64_t num_pages, int Hq, int Hkv, int D, int rot, int page_size,
                      int interleaved, int act_dtype, wlq_stream_t stream) {
    const char* fn = "wlq_rope_kv_write";
    clear_last_error();
    int rc;
    if (T < 0 || table_rows < 1) return fail(WLQ_ERR_INVALID_ARG, "%s: T=%lld, %lld table rows", fn, (long long)T, (long long)table_rows);
    if ((rc = bad_dtype(fn, act_dtype)) || (rc = bad_heads(fn, Hq, Hkv))) return rc;
    if (D < 16 || D > 256 || D % 16) return fail(WLQ_ERR_UNSUPPORTED, "%s: head size must be a multiple of 16 up to 256 (got %d)", fn, D);
    if (rot < 0 || rot > D || rot % 16) return fail(WLQ_ERR_UNSUPPORTED, "%s: the rotated part must be a multiple of 16 up to the head size %d (got %d)", fn, D, rot);
    if ((rc = bad_cache(fn, k_cache, v_cache, k_exp, v_exp, num_pages, page_size))) return rc;
    if (T == 0) return WLQ_OK;
    if (!positions || (rot && !cos_sin) || !slots) return fail(WLQ_ERR_INVALID_ARG, "%s: positions, cos_sin and slots are required", fn);
    if (!aligned16(cos_sin)) return fail(WLQ_ERR_ALIGNMENT, "%s: cos_sin must be 16-byte aligned", fn);
    if ((rc = bad_rows(fn, "q", q, q_tok, q_head)) || (rc = bad_rows(fn, "k", k, k_tok, k_head)) ||
        (rc = bad_rows(fn, "v", v, v_tok, v_head)) || (rc = bad_rows(fn, "q_out", q_out, qo_tok, qo_head)) ||
        (k_out && (rc = bad_rows(fn, "k_out", k_out, ko_tok, ko_head))))
        return rc;
    if (T > 0x7fffffff) return fail(WLQ_ERR_UNSUPPORTED, "%s: %lld tokens in one call", fn, (long long)T);
    if ((rc = require_sm100())) return rc;
    RopeParams p{};
    p.q = static_cast<const uint16_t*>(q);
    p.k = static_cast<const uint16_t*>(k);
    p.v = static_cast<const uint16_t*>(v);
    p.q_out = static_cast<uint16_t*>(q_out);
    p.k_out = static_cast<uint16_t*>(k_out);
    p.q_tok = q_tok, p.q_head = q_head, p.k_tok = k_tok, p.k_head = k_head, p.v_tok = v_tok, p.v_head = v_head;
    p.qo_tok = qo_tok, p.qo_head = qo_head, p.ko_tok = ko_tok, p.ko_head = ko_head;
    p.positions = positions;
    p.slots = slots;
    p.cos_sin = cos_sin;
    p.k_cache = k_cache, p.v_cache = v_cache, p.k_exp = k_exp, p.v_exp = v_exp;
    p.T = T, p.table_rows = table_rows, p.num_pages = num_pages;
    p.Hq = Hq, p.Hkv = Hkv, p.D = D, p.rot = rot, p.page_size = page_size, p.interleaved = interleaved != 0;
    return launch_rope_kv_write(p, act_dtype == WLQ_DTYPE_F16, k_exp != nullptr, static_cast<cudaStream_t>(stream));
}

int wlq_kv_read(const void* k_cache, const void* v_cache, const uint8_t* k_exp, const uint8_t* v_exp,
                const int32_t* block_table, const int32_t* cu_lens, void* k_out, void* v_out, int64_t T, int B,
                int64_t num_pages, int64_t table_cols, int Hkv, int D, int page_size, int act_dtype,
                wlq_stream_t stream) {
    const char* fn = "wlq_kv_read";
    clear_last_error();
    int rc;
    if (T < 0 || B < 0 || table_cols < 0) return fail(WLQ_ERR_INVALID_ARG, "%s: negative size", fn);
    if ((rc = bad_dtype(fn, act_dtype)) || (rc = bad_heads(fn, Hkv, Hkv))) return rc;
    if (D < 16 || D > 256 || D % 16 || Hkv * (D / 8) > 4096)
        return fail(WLQ_ERR_UNSUPPORTED, "%s: head size must be a multiple of 16 up to 256 (got %d, %d heads)", fn, D, Hkv);
    if ((rc = bad_cache(fn, k_cache, v_cache, k_exp, v_exp, num_pages, page_size))) return rc;
    if (T == 0) return WLQ_OK;
    if (B < 1 || !block_table || !cu_lens || !k_out || !v_out)
        return fail(WLQ_ERR_INVALID_ARG, "%s: block_table, cu_lens, k_out and v_out are required", fn);
    if (!aligned16(k_out) || !aligned16(v_out)) return fail(WLQ_ERR_ALIGNMENT, "%s: k_out and v_out must be 16-byte aligned", fn);
    if (T > 0x7fffffff) return fail(WLQ_ERR_UNSUPPORTED, "%s: %lld rows in one call", fn, (long long)T);
    if ((rc = require_sm100())) return rc;
    KvReadParams p{};
    p.k_cache = k_cache, p.v_cache = v_cache, p.k_exp = k_exp, p.v_exp = v_exp;
    p.table = block_table, p.cu = cu_lens;
    p.k_out = static_cast<uint16_t*>(k_out);
    p.v_out = static_cast<uint16_t*>(v_out);
    p.T = T, p.num_pages = num_pages, p.table_cols = table_cols;
    p.B = B, p.Hkv = Hkv, p.D = D, p.page_size = page_size;
    return launch_kv_read(p, act_dtype == WLQ_DTYPE_F16, k_exp != nullptr, static_cast<cudaStream_t>(stream));
}

int wlq_prompt_attention(const void* q, const void* k, const void* v, const int32_t* cu_seqlens, void* out,
                         int64_t q_tok, int64_t q_head, int64_t k_tok, int64_t k_head, int64_t v_tok, int64_t v_head,
                         int64_t o_tok, int64_t o_head, int64_t T, int B, int Hq, int Hkv, int D, float scale,
                         int causal, int act_dtype, wlq_stream_t stream) {
    const char* fn = "wlq_prompt_attention";
    clear_last_error();
    int rc;
    if (T < 0 || B < 0) return fail(WLQ_ERR_INVALID_ARG, "%s: negative size", fn);
    if ((rc = bad_dtype(fn, act_dtype)) || (rc = bad_heads(fn, Hq, Hkv))) return rc;
    if (D != 64 && D != 128) return fail(WLQ_ERR_UNSUPPORTED, "%s: head size must be 64 or 128 (got %d)", fn, D);
    if (Hq / Hkv > 128) return fail(WLQ_ERR_UNSUPPORTED, "%s: at most 128 query heads per kv head (got %d)", fn, Hq / Hkv);
    if (!(scale > 0.f) || !std::isfinite(scale)) return fail(WLQ_ERR_INVALID_ARG, "%s: scale must be positive and finite", fn);
    if (T == 0) return WLQ_OK;
    if (B < 1 || !cu_seqlens) return fail(WLQ_ERR_INVALID_ARG, "%s: cu_seqlens is required", fn);
    if ((rc = bad_rows(fn, "q", q, q_tok, q_head)) || (rc = bad_rows(fn, "k", k, k_tok, k_head)) ||
        (rc = bad_rows(fn, "v", v, v_tok, v_head)) || (rc = bad_rows(fn, "out", out, o_tok, o_head)))
        return rc;
    if (T * (Hq / Hkv) > 0x7fffffff) return fail(WLQ_ERR_UNSUPPORTED, "%s: %lld tokens in one call", fn, (long long)T);
    if ((rc = require_sm100())) return rc;
    AttnParams p{};
    p.q = static_cast<const uint16_t*>(q);
    p.k = static_cast<const uint16_t*>(k);
    p.v = static_cast<const uint16_t*>(v);
    p.out = static_cast<uint16_t*>(out);
    p.q_tok = q_tok, p.q_head = q_head, p.k_tok = k_tok, p.k_head = k_head, p.v_tok = v_tok, p.v_head = v_head;
    p.o_tok = o_tok, p.o_head = o_head;
    p.cu = cu_seqlens;
    p.T = T, p.B = B, p.Hq = Hq, p.Hkv = Hkv, p.G = Hq / Hkv, p.D = D, p.causal = causal != 0;
    p.scale_log2 = scale * 1.4426950408889634f;
    return launch_attention(p, act_dtype == WLQ_DTYPE_F16, static_cast<cudaStream_t>(stream));
}

size_t wlq_paged_attention_workspace_bytes(int Hq, int Hkv, int D, int max_q) {
    if (Hq < 1 || Hkv < 1 || D < 1 || max_q < 1) return 0;
    return attention_workspace_bytes(Hq, Hkv, D, max_q);
}

int wlq_paged_attention(const void* q, const void* k_cache, const void* v_cache, const uint8_t* k_exp,
                        const uint8_t* v_exp, const int32_t* block_table, const int32_t* kv_lens, const int32_t* cu_q,
                        void* out, int64_t q_tok, int64_t q_head, int64_t o_tok, int64_t o_head, int64_t T, int B,
                        int Hq, int Hkv, int D, int page_size, int64_t num_pages, int64_t table_cols, int max_q,
                        float scale, int act_dtype, void* workspace, size_t workspace_bytes, wlq_stream_t stream) {
    const char* fn = "wlq_paged_attention";
    clear_last_error();
    int rc;
    if (T < 0 || B < 0 || table_cols < 0 || max_q < 1) return fail(WLQ_ERR_INVALID_ARG, "%s: bad size", fn);
    if ((rc = bad_dtype(fn, act_dtype)) || (rc = bad_heads(fn, Hq, Hkv))) return rc;
    if (D != 64 && D != 128) return fail(WLQ_ERR_UNSUPPORTED, "%s: head size must be 64 or 128 (got %d)", fn, D);
    if (Hq / Hkv > 128) return fail(WLQ_ERR_UNSUPPORTED, "%s: at most 128 query heads per kv head (got %d)", fn, Hq / Hkv);
    if (!(scale > 0.f) || !std::isfinite(scale)) return fail(WLQ_ERR_INVALID_ARG, "%s: scale must be positive and finite", fn);
    if ((rc = bad_cache(fn, k_cache, v_cache, k_exp, v_exp, num_pages, page_size))) return rc;
    if (T == 0) return WLQ_OK;
    if (!block_table || !kv_lens) return fail(WLQ_ERR_INVALID_ARG, "%s: block_table and kv_lens are required", fn);
    if (B < 1) return fail(WLQ_ERR_INVALID_ARG, "%s: %lld tokens of 0 sequences", fn, (long long)T);
    if (!cu_q && (T != B || max_q != 1))
        return fail(WLQ_ERR_INVALID_ARG, "%s: without cu_q every sequence has one new token (T=%lld, B=%d, max_q=%d)", fn,
                    (long long)T, B, max_q);
    if ((rc = bad_rows(fn, "q", q, q_tok, q_head)) || (rc = bad_rows(fn, "out", out, o_tok, o_head))) return rc;
    if (T * (Hq / Hkv) > 0x7fffffff || table_cols * page_size > 0x7fffffff)
        return fail(WLQ_ERR_UNSUPPORTED, "%s: too many tokens for one call", fn);
    if ((int64_t)B * Hkv > (int64_t)WLQ_ATTENTION_ZERO_BYTES / 4)
        return fail(WLQ_ERR_UNSUPPORTED, "%s: %d sequences of %d kv heads (at most %u pairs)", fn, B, Hkv,
                    WLQ_ATTENTION_ZERO_BYTES / 4);
    // the few-row kernel counts the key tiles of all sequences and kv heads in 31 bits
    if ((int64_t)B * Hkv * ((table_cols * page_size + 63) / 64) > 0x7fffffff)
        return fail(WLQ_ERR_UNSUPPORTED, "%s: too many tokens for one call (%d sequences of up to %lld, %d kv heads)", fn, B,
                    (long long)(table_cols * page_size), Hkv);
    if (k_exp && (!aligned16(k_exp) || !aligned16(v_exp)))
        return fail(WLQ_ERR_ALIGNMENT, "%s: k_exp and v_exp must be 16-byte aligned", fn);
    if ((rc = require_sm100())) return rc;
    const size_t need = wlq_paged_attention_workspace_bytes(Hq, Hkv, D, max_q);
    if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
        return fail(WLQ_ERR_CAPACITY, "%s: needs a 16-byte aligned workspace of %zu bytes (got %zu)", fn, need,
                    workspace ? workspace_bytes : (size_t)0);
    AttnParams p{};
    p.q = static_cast<const uint16_t*>(q);
    p.out = static_cast<uint16_t*>(out);
    p.k_cache = k_cache, p.v_cache = v_cache, p.k_exp = k_exp, p.v_exp = v_exp;
    p.q_tok = q_tok, p.q_head = q_head, p.o_tok = o_tok, p.o_head = o_head;
    p.cu = cu_q, p.kv_lens = kv_lens, p.table = block_table;
    p.T = T, p.B = B, p.Hq = Hq, p.Hkv = Hkv, p.G = Hq / Hkv, p.D = D, p.page_size = page_size;
    p.log2_page = log2_of(page_size);
    p.num_pages = num_pages, p.table_cols = table_cols, p.causal = 1, p.max_q = max_q;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.ws = workspace, p.ws_bytes = workspace_bytes;
    return launch_attention(p, act_dtype == WLQ_DTYPE_F16, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
