// capi_serving.cpp -- extern "C" entry points of attention, the 4-bit cache of keys and
// values and the expert layer of few tokens: as in capi.cpp every argument is checked on
// the host before anything touches HIP.
#include "capi_checks.hpp"

#include <algorithm>

using w8a8::aligned;
using w8a8::check_heads;
using w8a8::check_kv4_cache;
using w8a8::fail;
using w8a8::hip_status;
using w8a8::valid_qmax;

namespace {

// Rows that go into or out of the cache; 0 where they are right.
int check_kv4_rows(const char* fn, const w8a8_kv4_cache* c, const void* k, const void* v,
                   const int32_t* slots, uint32_t tokens, uint32_t& ldk, uint32_t& ldv)
{
    if(const int rc = check_kv4_cache(fn, c)) return rc;
    if(tokens == 0) return 0;
    if(!k || !v || !slots) return fail(W8A8_ERROR_INVALID_VALUE, "%s: null pointer argument", fn);
    const uint64_t row = (uint64_t)c->kv_heads * c->head_dim;
    if(ldk == 0) ldk = (uint32_t)row;
    if(ldv == 0) ldv = (uint32_t)row;
    if(ldk < row || ldv < row)
        return fail(W8A8_ERROR_INVALID_VALUE,
                    "%s: ldk=%u / ldv=%u smaller than kv_heads * head_dim", fn, ldk, ldv);
    if(!aligned(k, 16) || !aligned(v, 16) || ldk % 8 || ldv % 8)
        return fail(W8A8_ERROR_NOT_SUPPORTED,
                    "%s: needs 16-byte aligned k, v and row strides of multiples of 8", fn);
    // a launch holds fewer than 2^32 threads: at most 256 a token, or two per 8 channels
    if((tokens + 8ull) * std::min<uint64_t>(256, row / 4) > 0xFFFFFFFFull)
        return fail(W8A8_ERROR_NOT_SUPPORTED, "%s: too many tokens in one call", fn);
    return 0;
}

} // namespace

extern "C" {

size_t w8a8_moe_ffn_decode_workspace_size(uint32_t tokens, uint32_t topk, uint32_t hidden,
                                          uint32_t inter)
{
    return w8a8::moe_ffn_decode_workspace_bytes(tokens, topk, hidden, inter);
}

int w8a8_moe_ffn_decode(const void* x, const void* logits, int logits_f16,
                        const float* smooth_scale, const int8_t* w_gate_up,
                        const float* sb_gate_up, const float* smooth_scale_down,
                        const int8_t* w_down, const float* sb_down, void* out, uint32_t tokens,
                        uint32_t hidden, uint32_t inter, uint32_t experts, uint32_t topk,
                        float quant_max, uint32_t ldx, uint32_t ldo, void* workspace,
                        size_t ws_bytes, hipStream_t stream)
{
    const char* fn = "w8a8_moe_ffn_decode";
    if(tokens == 0) return hip_status(hipSuccess, fn);
    if(!x || !logits || !smooth_scale || !w_gate_up || !sb_gate_up || !w_down || !sb_down || !out
       || !workspace)
        return fail(W8A8_ERROR_INVALID_VALUE, "%s: null pointer argument", fn);
    if(hidden == 0 || inter == 0 || experts == 0 || topk == 0)
        return fail(W8A8_ERROR_INVALID_VALUE, "%s: hidden, inter, experts and topk must be > 0",
                    fn);
    if(topk > experts)
        return fail(W8A8_ERROR_INVALID_VALUE, "%s: topk=%u > experts=%u", fn, topk, experts);
    if(tokens > W8A8_MOE_DECODE_MAX_TOKENS || (uint64_t)tokens * hidden > W8A8_MOE_DECODE_MAX_VALUES
       || experts > 4096 || topk > 32)
        return fail(W8A8_ERROR_NOT_SUPPORTED,
                    "%s: needs tokens <= %u, tokens * hidden <= %u, experts <= 4096, topk <= 32 "
                    "(tokens=%u hidden=%u experts=%u topk=%u)",
                    fn, W8A8_MOE_DECODE_MAX_TOKENS, W8A8_MOE_DECODE_MAX_VALUES, tokens, hidden,
                    experts, topk);
    if(hidden % 16 != 0 || inter % 16 != 0 || hidden > 32768 || inter > 32768)
        return fail(W8A8_ERROR_NOT_SUPPORTED,
                    "%s: needs hidden and inter multiples of 16, at most 32768 (hidden=%u "
                    "inter=%u)",
                    fn, hidden, inter);
    if(!valid_qmax(quant_max))
        return fail(W8A8_ERROR_INVALID_VALUE, "%s: quant_max must be in (0, 127]", fn);
    if(ldx == 0) ldx = hidden;
    if(ldo == 0) ldo = hidden;
    if(ldx < hidden || ldo < hidden)
        return fail(W8A8_ERROR_INVALID_VALUE, "%s: ldx=%u / ldo=%u smaller than hidden=%u", fn, ldx,
                    ldo, hidden);
    if(!aligned(x, 16) || ldx % 8 != 0 || !aligned(smooth_scale, 16) || !aligned(w_gate_up, 16)
       || !aligned(smooth_scale_down, 16) || !aligned(w_down, 16) || !aligned(sb_gate_up, 16)
       || !aligned(sb_down, 16) || !aligned(out, 2))
        return fail(W8A8_ERROR_NOT_SUPPORTED,
                    "%s: needs 16-byte aligned x, smooth scales, weights and weight scales, ldx "
                    "%% 8 == 0",
                    fn);
    if(!aligned(workspace, 256))
        return fail(W8A8_ERROR_INVALID_VALUE, "%s: workspace must be 256-byte aligned", fn);
    const size_t need = w8a8::moe_ffn_decode_workspace_bytes(tokens, topk, hidden, inter);
    if(ws_bytes < need)
        return fail(W8A8_ERROR_INVALID_VALUE, "%s: workspace of %zu bytes, %zu needed", fn, ws_bytes,
                    need);
    w8a8::MoeDecodeArgs a{static_cast<const uint16_t*>(x),
                          logits,
                          smooth_scale,
                          w_gate_up,
                          sb_gate_up,
                          smooth_scale_down,
                          w_down,
                          sb_down,
                          static_cast<uint16_t*>(out),
                          tokens,
                          hidden,
                          inter,
                          experts,
                          topk,
                          ldx,
                          ldo,
                          quant_max,
                          workspace};
    return hip_status(w8a8::launch_moe_ffn_decode(a, logits_f16 != 0, stream), fn);
}

int w8a8_attention(const void* q, const void* k, const void* v, void* out,
                   const int32_t* seq_starts, uint32_t seqs, uint32_t tokens, uint32_t heads,
                   uint32_t kv_heads, uint32_t head_dim, uint32_t ldq, uint32_t ldk,
                   uint32_t ldv, uint32_t ldo, float scale, hipStream_t stream)
{
    const char* fn = "w8a8_attention";
    if(const int rc = check_heads(fn, heads, kv_heads, head_dim, scale)) return rc;
    if(tokens == 0 || seqs == 0) return hip_status(hipSuccess, fn);
    if(!q || !k || !v || !out || !seq_starts)
        return fail(W8A8_ERROR_INVALID_VALUE, "%s: null pointer argument", fn);
    if(tokens > 0x7FFFFFFFu || seqs > 0x7FFFFFFu)
        return fail(W8A8_ERROR_NOT_SUPPORTED, "%s: needs tokens < 2^31, seqs < 2^27", fn);
    const uint64_t row = (uint64_t)heads * head_dim, kv_row = (uint64_t)kv_heads * head_dim;
    if(ldq < row || ldo < row || ldk < kv_row || ldv < kv_row)
        return fail(W8A8_ERROR_INVALID_VALUE,
                    "%s: ldq=%u, ldo=%u must be >= heads * head_dim, ldk=%u, ldv=%u >= kv_heads * "
                    "head_dim",
                    fn, ldq, ldo, ldk, ldv);
    if(!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16) || ldq % 8
       || ldk % 8 || ldv % 8 || ldo % 8)
        return fail(W8A8_ERROR_NOT_SUPPORTED,
                    "%s: needs 16-byte aligned q, k, v, out and row strides of multiples of 8", fn);
    // a block of 256 threads per (128 rows, head), and a launch of fewer than 2^32 threads
    if(((uint64_t)tokens / 128 + seqs) * heads > 0xFFFFFFull || ldk > 0x1000000u
       || ldv > 0x1000000u || ldq > 0x1000000u || ldo > 0x1000000u)
        return fail(W8A8_ERROR_NOT_SUPPORTED, "%s: too many tokens, sequences or columns", fn);
    w8a8::AttentionArgs a{static_cast<const uint16_t*>(q),
                          static_cast<const uint16_t*>(k),
                          static_cast<const uint16_t*>(v),
                          static_cast<uint16_t*>(out),
                          seq_starts,
                          seqs,
                          tokens,
                          heads,
                          kv_heads,
                          head_dim,
                          ldq,
                          ldk,
                          ldv,
                          ldo,
                          scale};
    return hip_status(w8a8::launch_attention(a, stream), fn);
}

int w8a8_kv4_store(const void* k, const void* v, const int32_t* slots, uint32_t tokens,
                   uint32_t ldk, uint32_t ldv, const w8a8_kv4_cache* cache, hipStream_t stream)
{
    const char* fn = "w8a8_kv4_store";
    if(const int rc = check_kv4_rows(fn, cache, k, v, slots, tokens, ldk, ldv)) return rc;
    if(tokens == 0) return hip_status(hipSuccess, fn);
    return hip_status(w8a8::launch_kv4_store(*cache, {slots, tokens, ldk, ldv},
                                             static_cast<const uint16_t*>(k),
                                             static_cast<const uint16_t*>(v), stream),
                      fn);
}

int w8a8_kv4_load(void* k, void* v, const int32_t* slots, uint32_t tokens, uint32_t ldk,
                  uint32_t ldv, const w8a8_kv4_cache* cache, hipStream_t stream)
{
    const char* fn = "w8a8_kv4_load";
    if(const int rc = check_kv4_rows(fn, cache, k, v, slots, tokens, ldk, ldv)) return rc;
    if(tokens == 0) return hip_status(hipSuccess, fn);
    return hip_status(w8a8::launch_kv4_load(*cache, {slots, tokens, ldk, ldv},
                                            static_cast<uint16_t*>(k), static_cast<uint16_t*>(v),
                                            stream),
                      fn);
}

size_t w8a8_attention_kv4_workspace_size(uint32_t seqs, uint32_t heads, uint32_t kv_heads,
                                         uint32_t head_dim, uint32_t max_len)
{
    if(kv_heads == 0 || heads == 0 || heads % kv_heads != 0) return 0;
    return w8a8::attention_kv4_workspace_bytes(seqs, heads, kv_heads, head_dim, max_len);
}

int w8a8_attention_kv4(const void* q, const w8a8_kv4_cache* cache, const int32_t* block_table,
                       uint32_t table_cols, uint32_t table_ld, const int32_t* seq_lens, void* out,
                       uint32_t seqs, uint32_t heads, uint32_t ldq, uint32_t ldo, float scale,
                       void* workspace, size_t ws_bytes, hipStream_t stream)
{
    const char* fn = "w8a8_attention_kv4";
    if(const int rc = w8a8::check_attention_kv4(fn, q, cache, block_table, table_cols, table_ld,
                                                seq_lens, out, seqs, heads, ldq, ldo, scale,
                                                workspace))
        return rc;
    if(seqs == 0) return hip_status(hipSuccess, fn);
    w8a8::AttentionKv4Args a{static_cast<const uint16_t*>(q),
                             static_cast<uint16_t*>(out),
                             block_table,
                             seq_lens,
                             seqs,
                             heads,
                             ldq,
                             ldo,
                             table_cols,
                             table_ld,
                             scale,
                             workspace,
                             workspace ? ws_bytes : 0};
    return hip_status(w8a8::launch_attention_kv4(*cache, a, stream), fn);
}

} // extern "C"
