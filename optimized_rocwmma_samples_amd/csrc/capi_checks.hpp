// capi_checks.hpp -- argument checks that the entry points of attention and of the 4-bit
// cache share.
#pragma once

#include "../../include/w8a8.h"
#include "w8a8_internal.hpp"

#include <cmath>

namespace w8a8 {

inline bool aligned(const void* p, uintptr_t bytes)
{
    return reinterpret_cast<uintptr_t>(p) % bytes == 0;
}

// The head counts and scale of an attention call; 0 where they are right.
inline int check_heads(const char* fn, uint32_t heads, uint32_t kv_heads, uint32_t head_dim,
                       float scale)
{
    if(heads == 0 || kv_heads == 0 || heads % kv_heads != 0)
        return fail(W8A8_ERROR_INVALID_VALUE,
                    "%s: kv_heads must divide heads, both > 0 (heads=%u kv_heads=%u)", fn, heads,
                    kv_heads);
    if(head_dim != 64 && head_dim != 128)
        return fail(W8A8_ERROR_NOT_SUPPORTED, "%s: head_dim must be 64 or 128, got %u", fn,
                    head_dim);
    if(!(std::isfinite(scale) && scale > 0.f))
        return fail(W8A8_ERROR_INVALID_VALUE, "%s: scale must be finite and > 0, got %g", fn,
                    (double)scale);
    return 0;
}

// The cache descriptor; 0 where it is right.
inline int check_kv4_cache(const char* fn, const w8a8_kv4_cache* c)
{
    if(!c || !c->k_codes || !c->v_codes || !c->k_scales || !c->v_scales)
        return fail(W8A8_ERROR_INVALID_VALUE, "%s: null pointer in the cache descriptor", fn);
    if(c->pages == 0 || c->kv_heads == 0)
        return fail(W8A8_ERROR_INVALID_VALUE, "%s: pages and kv_heads must be > 0", fn);
    if(c->head_dim != 64 && c->head_dim != 128)
        return fail(W8A8_ERROR_NOT_SUPPORTED, "%s: head_dim must be 64 or 128, got %u", fn,
                    c->head_dim);
    if((c->group != 32 && c->group != 64 && c->group != 128) || c->group > c->head_dim)
        return fail(W8A8_ERROR_NOT_SUPPORTED,
                    "%s: group must be 32, 64 or 128 and at most head_dim, got %u", fn, c->group);
    if(c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)) != 0)
        return fail(W8A8_ERROR_NOT_SUPPORTED,
                    "%s: page_size must be a power of two in 16..1024, got %u", fn, c->page_size);
    if((uint64_t)c->pages * c->page_size > 0x7FFFFFFFull || c->kv_heads > 65535)
        return fail(W8A8_ERROR_NOT_SUPPORTED,
                    "%s: needs pages * page_size < 2^31 and kv_heads < 65536", fn);
    if(!aligned(c->k_codes, 16) || !aligned(c->v_codes, 16) || !aligned(c->k_scales, 16)
       || !aligned(c->v_scales, 16))
        return fail(W8A8_ERROR_NOT_SUPPORTED, "%s: cache buffers must be 16-byte aligned", fn);
    return 0;
}

// The arguments of an attention of single tokens over the cache; 0 where they are right.
inline int check_attention_kv4(const char* fn, const void* q, const w8a8_kv4_cache* cache,
                               const int32_t* block_table, uint32_t table_cols, uint32_t table_ld,
                               const int32_t* seq_lens, const void* out, uint32_t seqs,
                               uint32_t heads, uint32_t ldq, uint32_t ldo, float scale,
                               const void* workspace)
{
    if(const int rc = check_kv4_cache(fn, cache)) return rc;
    if(const int rc = check_heads(fn, heads, cache->kv_heads, cache->head_dim, scale)) return rc;
    if(seqs == 0) return 0;
    if(!q || !out || !seq_lens || (!block_table && table_cols != 0))
        return fail(W8A8_ERROR_INVALID_VALUE, "%s: null pointer argument", fn);
    const uint64_t row = (uint64_t)heads * cache->head_dim;
    if(ldq < row || ldo < row || table_ld < table_cols)
        return fail(W8A8_ERROR_INVALID_VALUE,
                    "%s: ldq=%u, ldo=%u must be >= heads * head_dim, table_ld=%u >= table_cols=%u",
                    fn, ldq, ldo, table_ld, table_cols);
    if(!aligned(q, 16) || !aligned(out, 16) || ldq % 8 || ldo % 8)
        return fail(W8A8_ERROR_NOT_SUPPORTED,
                    "%s: needs 16-byte aligned q, out and row strides of multiples of 8", fn);
    if((uint64_t)table_cols * cache->page_size > 0x7FFFFFFFull
       || (uint64_t)seqs * heads > 0xFFFFFFull)
        return fail(W8A8_ERROR_NOT_SUPPORTED,
                    "%s: needs table_cols * page_size < 2^31 and seqs * heads < 2^24", fn);
    // the chunks of 64 tokens of all sequences are counted in 31 bits
    if(((uint64_t)table_cols * cache->page_size / 64 + 1) * seqs * heads > 0x7FFFFFFFull)
        return fail(W8A8_ERROR_NOT_SUPPORTED,
                    "%s: needs seqs * heads * (table_cols * page_size / 64 + 1) < 2^31", fn);
    if(!aligned(workspace, 16))
        return fail(W8A8_ERROR_INVALID_VALUE, "%s: workspace must be 16-byte aligned", fn);
    return 0;
}

} // namespace w8a8
