// capi_paged.cpp -- extern "C" entry points of the paged 4-bit cache in service: pages handed
// out and taken back, page keys and the pages that suit a query, attention of chunks over the
// cache and over selected pages.  As in capi.cpp every argument is checked on the host
// before anything touches HIP.
#include "capi_checks.hpp"

using w8a8::aligned;
using w8a8::check_heads;
using w8a8::check_kv4_cache;
using w8a8::fail;
using w8a8::hip_status;

namespace {

// Sequences, their block table and the size of its pages; 0 where they are right.
int check_table(const char* fn, uint32_t seqs, uint32_t table_cols, uint32_t table_ld,
                uint32_t page_size)
{
    if(table_ld < table_cols)
        return fail(W8A8_ERROR_INVALID_VALUE, "%s: table_ld=%u smaller than table_cols=%u", fn,
                    table_ld, table_cols);
    if(page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)) != 0)
        return fail(W8A8_ERROR_NOT_SUPPORTED,
                    "%s: page_size must be a power of two in 16..1024, got %u", fn, page_size);
    if((uint64_t)table_cols * page_size > 0x7FFFFFFFull || seqs > 0x7FFFFFFu)
        return fail(W8A8_ERROR_NOT_SUPPORTED,
                    "%s: needs table_cols * page_size < 2^31 and seqs < 2^27", fn);
    return 0;
}

// Page keys; 0 where they are right.
int check_page_keys(const char* fn, const w8a8_kv4_page_keys* k)
{
    if(!k || !k->codes || !k->scales)
        return fail(W8A8_ERROR_INVALID_VALUE, "%s: null pointer in the page keys", fn);
    if(k->pages == 0 || k->kv_heads == 0 || k->pages > 0x7FFFFFFFu || k->kv_heads > 65535)
        return fail(W8A8_ERROR_INVALID_VALUE, "%s: needs 0 < pages < 2^31, 0 < kv_heads < 65536",
                    fn);
    if(k->head_dim != 64 && k->head_dim != 128)
        return fail(W8A8_ERROR_NOT_SUPPORTED, "%s: head_dim must be 64 or 128, got %u", fn,
                    k->head_dim);
    if(!aligned(k->codes, 16) || !aligned(k->scales, 16))
        return fail(W8A8_ERROR_NOT_SUPPORTED, "%s: page keys must be 16-byte aligned", fn);
    return 0;
}

} // namespace

extern "C" {

int w8a8_kv4_extend(const int32_t* new_tokens, const int32_t* seq_lens, uint32_t seqs,
                    int32_t* block_table, uint32_t table_cols, uint32_t table_ld,
                    const int32_t* free_pages, uint32_t free_capacity, const int32_t* free_count,
                    uint32_t page_size, int32_t* slots, uint32_t tokens, int32_t* seq_starts,
                    int32_t* lens_out, int32_t* count_out, hipStream_t stream)
{
    const char* fn = "w8a8_kv4_extend";
    if(const int rc = check_table(fn, seqs, table_cols, table_ld, page_size)) return rc;
    if(!free_count || !seq_starts || !count_out || (!free_pages && free_capacity != 0)
       || (!slots && tokens != 0)
       || (seqs != 0
           && (!new_tokens || !seq_lens || !lens_out || (!block_table && table_cols != 0))))
        return fail(W8A8_ERROR_INVALID_VALUE, "%s: null pointer argument", fn);
    if(tokens > 0x7FFFFFFEu || free_capacity > 0x7FFFFFFFu)
        return fail(W8A8_ERROR_NOT_SUPPORTED, "%s: needs tokens and free_capacity < 2^31 - 1", fn);
    w8a8::Kv4ExtendArgs a{};
    a.fresh      = new_tokens;
    a.lens       = seq_lens;
    a.table      = block_table;
    a.free       = free_pages;
    a.count      = free_count;
    a.slots      = slots;
    a.starts     = seq_starts;
    a.lens_out   = lens_out;
    a.count_out  = count_out;
    a.seqs       = seqs;
    a.tokens     = tokens;
    a.table_cols = table_cols;
    a.table_ld   = table_ld;
    a.capacity   = free_capacity;
    a.page_shift = (uint32_t)__builtin_ctz(page_size);
    return hip_status(w8a8::launch_kv4_extend(a, stream), fn);
}

int w8a8_kv4_trim(const int32_t* keep, const int32_t* seq_lens, uint32_t seqs,
                  const int32_t* block_table, uint32_t table_cols, uint32_t table_ld,
                  int32_t* free_pages, uint32_t free_capacity, const int32_t* free_count,
                  uint32_t page_size, int32_t* lens_out, int32_t* count_out, hipStream_t stream)
{
    const char* fn = "w8a8_kv4_trim";
    if(const int rc = check_table(fn, seqs, table_cols, table_ld, page_size)) return rc;
    if(!free_count || !count_out || (!free_pages && free_capacity != 0)
       || (seqs != 0 && (!keep || !seq_lens || !lens_out || (!block_table && table_cols != 0))))
        return fail(W8A8_ERROR_INVALID_VALUE, "%s: null pointer argument", fn);
    // a block counts the pages of all sequences in 32 bits
    if(free_capacity > 0x7FFFFFFFu || (uint64_t)seqs * table_cols > 0x7FFFFFFFull)
        return fail(W8A8_ERROR_NOT_SUPPORTED,
                    "%s: needs free_capacity and seqs * table_cols < 2^31", fn);
    w8a8::Kv4TrimArgs a{};
    a.keep       = keep;
    a.lens       = seq_lens;
    a.table      = block_table;
    a.free       = free_pages;
    a.count      = free_count;
    a.lens_out   = lens_out;
    a.count_out  = count_out;
    a.seqs       = seqs;
    a.table_cols = table_cols;
    a.table_ld   = table_ld;
    a.capacity   = free_capacity;
    a.page_shift = (uint32_t)__builtin_ctz(page_size);
    return hip_status(w8a8::launch_kv4_trim(a, stream), fn);
}

int w8a8_kv4_summarize(const w8a8_kv4_cache* cache, const w8a8_kv4_page_keys* keys,
                       const int32_t* block_table, uint32_t table_cols, uint32_t table_ld,
                       const int32_t* seq_lens, const int32_t* seq_starts, uint32_t seqs,
                       uint32_t tokens, hipStream_t stream)
{
    const char* fn = "w8a8_kv4_summarize";
    if(const int rc = check_kv4_cache(fn, cache)) return rc;
    if(const int rc = check_page_keys(fn, keys)) return rc;
    if(keys->pages != cache->pages || keys->kv_heads != cache->kv_heads
       || keys->head_dim != cache->head_dim)
        return fail(W8A8_ERROR_INVALID_VALUE,
                    "%s: the page keys are not this cache's (pages, kv_heads, head_dim)", fn);
    if(const int rc = check_table(fn, seqs, table_cols, table_ld, cache->page_size)) return rc;
    if(seqs == 0 || tokens == 0 || table_cols == 0) return hip_status(hipSuccess, fn);
    if(!block_table || !seq_lens || !seq_starts)
        return fail(W8A8_ERROR_INVALID_VALUE, "%s: null pointer argument", fn);
    // a wave of 64 threads per page and key head, and a launch of fewer than 2^32 threads
    if(tokens > 0x7FFFFFFFu
       || w8a8::kv4_touched_pages(tokens, seqs, cache->page_size) * cache->kv_heads > 0x3FFFFF0ull)
        return fail(W8A8_ERROR_NOT_SUPPORTED, "%s: too many tokens or sequences in one call", fn);
    w8a8::Kv4SummarizeArgs a{};
    a.table      = block_table;
    a.lens       = seq_lens;
    a.starts     = seq_starts;
    a.codes      = keys->codes;
    a.scales     = keys->scales;
    a.seqs       = seqs;
    a.tokens     = tokens;
    a.table_cols = table_cols;
    a.table_ld   = table_ld;
    return hip_status(w8a8::launch_kv4_summarize(*cache, a, stream), fn);
}

int w8a8_kv4_page_keys_load(const w8a8_kv4_page_keys* keys, const int32_t* pages, uint32_t count,
                            float* out, hipStream_t stream)
{
    const char* fn = "w8a8_kv4_page_keys_load";
    if(const int rc = check_page_keys(fn, keys)) return rc;
    if(count == 0) return hip_status(hipSuccess, fn);
    if(!pages || !out) return fail(W8A8_ERROR_INVALID_VALUE, "%s: null pointer argument", fn);
    if(!aligned(out, 16))
        return fail(W8A8_ERROR_NOT_SUPPORTED, "%s: needs a 16-byte aligned out", fn);
    if((uint64_t)count * keys->kv_heads * (keys->head_dim / 4) > 0xFFFFFF00ull)
        return fail(W8A8_ERROR_NOT_SUPPORTED, "%s: too many pages in one call", fn);
    w8a8::Kv4PageKeysArgs a{keys->codes, keys->scales, pages,          out,
                            count,       keys->pages,  keys->kv_heads, keys->head_dim};
    return hip_status(w8a8::launch_kv4_page_keys(a, stream), fn);
}

size_t w8a8_kv4_select_workspace_size(uint32_t seqs, uint32_t kv_heads, uint32_t table_cols,
                                      uint32_t keep)
{
    return w8a8::kv4_select_workspace_bytes(seqs, kv_heads, table_cols, keep);
}

int w8a8_kv4_select(const void* q, const w8a8_kv4_page_keys* keys, const int32_t* block_table,
                    uint32_t table_cols, uint32_t table_ld, const int32_t* seq_lens,
                    uint32_t page_size, int32_t* chosen, uint32_t keep, int32_t* lens_out,
                    uint32_t seqs, uint32_t heads, uint32_t ldq, void* workspace, size_t ws_bytes,
                    hipStream_t stream)
{
    const char* fn = "w8a8_kv4_select";
    if(const int rc = check_page_keys(fn, keys)) return rc;
    if(const int rc = check_heads(fn, heads, keys->kv_heads, keys->head_dim, 1.f)) return rc;
    if(const int rc = check_table(fn, seqs, table_cols, table_ld, page_size)) return rc;
    if(keep == 0) return fail(W8A8_ERROR_INVALID_VALUE, "%s: keep must be > 0", fn);
    if(seqs == 0) return hip_status(hipSuccess, fn);
    if(!q || !seq_lens || !chosen || !lens_out || (!block_table && table_cols != 0))
        return fail(W8A8_ERROR_INVALID_VALUE, "%s: null pointer argument", fn);
    if(ldq < (uint64_t)heads * keys->head_dim)
        return fail(W8A8_ERROR_INVALID_VALUE, "%s: ldq=%u smaller than heads * head_dim", fn, ldq);
    // a block of 1024 threads per sequence and key head, one of 256 per 256 pages of them,
    // and a launch of fewer than 2^32 threads
    const uint64_t units = (uint64_t)seqs * keys->kv_heads;
    if(units > 0x3FFFFFull || units * (table_cols / 256ull + 1) > 0xFFFFFFull
       || units * keep > 0x7FFFFFFFull)
        return fail(W8A8_ERROR_NOT_SUPPORTED,
                    "%s: too many sequences, key heads or columns in one call", fn);
    const size_t need = w8a8::kv4_select_workspace_bytes(seqs, keys->kv_heads, table_cols, keep);
    if(need != 0 && (!workspace || ws_bytes < need || !aligned(workspace, 16)))
        return fail(W8A8_ERROR_INVALID_VALUE,
                    "%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", fn, need,
                    workspace ? ws_bytes : 0);
    w8a8::Kv4SelectArgs a{};
    a.q          = static_cast<const uint16_t*>(q);
    a.codes      = keys->codes;
    a.scales     = keys->scales;
    a.table      = block_table;
    a.lens       = seq_lens;
    a.chosen     = chosen;
    a.lens_out   = lens_out;
    a.seqs       = seqs;
    a.heads      = heads;
    a.kv_heads   = keys->kv_heads;
    a.head_dim   = keys->head_dim;
    a.ldq        = ldq;
    a.table_cols = table_cols;
    a.table_ld   = table_ld;
    a.keep       = keep;
    a.page_shift = (uint32_t)__builtin_ctz(page_size);
    a.pages      = keys->pages;
    a.ws         = workspace;
    return hip_status(w8a8::launch_kv4_select(a, stream), fn);
}

int w8a8_attention_kv4_selected(const void* q, const w8a8_kv4_cache* cache,
                                const int32_t* block_tables, uint32_t table_cols,
                                const int32_t* seq_lens, void* out, uint32_t seqs, uint32_t heads,
                                uint32_t ldq, uint32_t ldo, float scale, void* workspace,
                                size_t ws_bytes, hipStream_t stream)
{
    const char* fn = "w8a8_attention_kv4_selected";
    if(const int rc = w8a8::check_attention_kv4(fn, q, cache, block_tables, table_cols, table_cols,
                                                seq_lens, out, seqs, heads, ldq, ldo, scale,
                                                workspace))
        return rc;
    if(seqs == 0) return hip_status(hipSuccess, fn);
    if((uint64_t)table_cols * cache->kv_heads > 0xFFFFFFFFull)
        return fail(W8A8_ERROR_NOT_SUPPORTED, "%s: needs table_cols * kv_heads < 2^32", fn);
    w8a8::AttentionKv4Args a{static_cast<const uint16_t*>(q),
                             static_cast<uint16_t*>(out),
                             block_tables,
                             seq_lens,
                             seqs,
                             heads,
                             ldq,
                             ldo,
                             table_cols,
                             table_cols * cache->kv_heads,
                             scale,
                             workspace,
                             workspace ? ws_bytes : 0,
                             table_cols};
    return hip_status(w8a8::launch_attention_kv4(*cache, a, stream), fn);
}

size_t w8a8_attention_kv4_chunks_workspace_size(const w8a8_kv4_cache* cache, uint32_t seqs,
                                                uint32_t tokens, uint32_t heads,
                                                uint32_t table_cols, uint32_t max_new)
{
    if(check_kv4_cache("w8a8_attention_kv4_chunks_workspace_size", cache) != 0 || heads == 0
       || heads % cache->kv_heads != 0)
        return 0;
    return w8a8::attention_kv4_chunks_workspace_bytes(*cache, seqs, tokens, heads, table_cols,
                                                      max_new);
}

int w8a8_attention_kv4_chunks(const void* q, const w8a8_kv4_cache* cache,
                              const int32_t* block_table, uint32_t table_cols, uint32_t table_ld,
                              const int32_t* seq_lens, const int32_t* seq_starts, void* out,
                              uint32_t seqs, uint32_t tokens, uint32_t heads, uint32_t max_new,
                              uint32_t ldq, uint32_t ldo, float scale, void* workspace,
                              size_t ws_bytes, hipStream_t stream)
{
    const char* fn = "w8a8_attention_kv4_chunks";
    if(const int rc = check_kv4_cache(fn, cache)) return rc;
    if(const int rc = check_heads(fn, heads, cache->kv_heads, cache->head_dim, scale)) return rc;
    if(const int rc = check_table(fn, seqs, table_cols, table_ld, cache->page_size)) return rc;
    if(seqs == 0 || tokens == 0) return hip_status(hipSuccess, fn);
    if(!q || !out || !seq_lens || !seq_starts || (!block_table && table_cols != 0))
        return fail(W8A8_ERROR_INVALID_VALUE, "%s: null pointer argument", fn);
    const uint64_t row = (uint64_t)heads * cache->head_dim;
    if(ldq < row || ldo < row)
        return fail(W8A8_ERROR_INVALID_VALUE, "%s: ldq=%u, ldo=%u must be >= heads * head_dim", fn,
                    ldq, ldo);
    if(!aligned(q, 16) || !aligned(out, 16) || ldq % 8 || ldo % 8)
        return fail(W8A8_ERROR_NOT_SUPPORTED,
                    "%s: needs 16-byte aligned q, out and row strides of multiples of 8", fn);
    // steps of 128 keys of 32 rows, counted in 31 bits; a sequence's rows likewise
    const uint64_t some  = tokens < seqs ? tokens : seqs;
    const uint64_t tiles = (uint64_t)tokens * heads / 32 + some * cache->kv_heads;
    if(tokens > 0x7FFFFFFFu || (uint64_t)tokens * heads > 0x7FFFFFFFull
       || tiles * ((uint64_t)table_cols * cache->page_size / 128 + 1) > 0x7FFFFFFFull)
        return fail(W8A8_ERROR_NOT_SUPPORTED, "%s: too many tokens, heads or columns in one call",
                    fn);
    const size_t need = w8a8::attention_kv4_chunks_workspace_bytes(*cache, seqs, tokens, heads,
                                                                   table_cols, max_new);
    if(need != 0 && (!workspace || ws_bytes < need || !aligned(workspace, 256)))
        return fail(W8A8_ERROR_INVALID_VALUE,
                    "%s: needs a 256-byte aligned workspace of %zu bytes, got %zu", fn, need,
                    workspace ? ws_bytes : 0);
    w8a8::ChunkArgs a{};
    a.q          = static_cast<const uint16_t*>(q);
    a.out        = static_cast<uint16_t*>(out);
    a.table      = block_table;
    a.lens       = seq_lens;
    a.starts     = seq_starts;
    a.seqs       = seqs;
    a.tokens     = tokens;
    a.heads      = heads;
    a.ldq        = ldq;
    a.ldo        = ldo;
    a.table_cols = table_cols;
    a.table_ld   = table_ld;
    a.max_new    = max_new == 0 || max_new > tokens ? tokens : max_new;
    a.scale      = scale;
    a.ws         = workspace;
    return hip_status(w8a8::launch_attention_kv4_chunks(*cache, a, stream), fn);
}

} // extern "C"
