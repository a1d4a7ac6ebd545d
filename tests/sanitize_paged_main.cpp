// Driver of the host side of the paged 4-bit cache in service for the sanitizer build of
// test_sanitizers_paged_cpu.py: every entry point with arguments its checks reject, its size
// queries over a range of shapes, and the calls that have nothing to do.  Nothing here
// reaches a kernel launch, and no pointer below is dereferenced but the descriptors'.  Prints
// "OK <calls>" on success.
#include "../include/w8a8.h"

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>

static char g_msg[512];
static int  g_calls = 0;

// what capi.cpp holds for all entry points
namespace w8a8 {
int fail(int code, const char* fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_msg, sizeof(g_msg), fmt, ap);
    va_end(ap);
    return code;
}
int hip_status(hipError_t e, const char* what)
{
    return e == hipSuccess ? 0 : fail((int)e, "%s", what);
}
} // namespace w8a8

static void expect(int rc, int want, const char* what, int line)
{
    ++g_calls;
    if(rc != want || (want != 0 && g_msg[0] == '\0')) {
        std::printf("FAIL line %d (%s): rc=%d, %d expected\n", line, what, rc, want);
        std::exit(1);
    }
    g_msg[0] = '\0';
}
#define INVALID(call) expect((call), W8A8_ERROR_INVALID_VALUE, #call, __LINE__)
#define UNSUPPORTED(call) expect((call), W8A8_ERROR_NOT_SUPPORTED, #call, __LINE__)
#define DONE(call) expect((call), W8A8_SUCCESS, #call, __LINE__)

int main()
{
    void*       P  = reinterpret_cast<void*>(0x100000);
    void*       O  = reinterpret_cast<void*>(0x100008); // off the 16-byte alignment
    int32_t*    I  = static_cast<int32_t*>(P);
    uint8_t*    B  = static_cast<uint8_t*>(P);
    hipStream_t st = nullptr;

    const w8a8_kv4_cache     cache = {B, B, P, P, 4, 32, 2, 64, 32};
    const w8a8_kv4_page_keys keys  = {static_cast<int8_t*>(P), static_cast<float*>(P), 4, 2, 64};

    // ---- size queries -------------------------------------------------------
    size_t sink = 0;
    for(uint32_t s : {0u, 1u, 48u, 65536u})
        for(uint32_t t : {0u, 1u, 300u, 65536u, 0x7FFFFFFFu})
            for(uint32_t h : {0u, 2u, 6u, 64u, 130u})
                for(uint32_t cols : {0u, 1u, 5u, 4096u, 0x3FFFFFFu})
                    for(uint32_t m : {0u, 1u, 300u, 0xFFFFFFFFu}) {
                        sink += w8a8_attention_kv4_chunks_workspace_size(&cache, s, t, h, cols, m);
                        sink += w8a8_kv4_select_workspace_size(s, h, cols, m);
                    }
    if(sink == 0 || w8a8_attention_kv4_chunks_workspace_size(nullptr, 1, 1, 2, 1, 0) != 0) return 1;
    g_msg[0] = '\0';

    // ---- pages --------------------------------------------------------------
    auto extend = [&](const int32_t* fresh, uint32_t seqs, uint32_t cols, uint32_t ld, uint32_t cap,
                      uint32_t page, uint32_t tokens, int32_t* count) {
        return w8a8_kv4_extend(fresh, I, seqs, I, cols, ld, I, cap, I, page, I, tokens, I, I, count,
                               st);
    };
    INVALID(extend(nullptr, 2, 3, 3, 9, 16, 4, I));
    INVALID(extend(I, 2, 3, 2, 9, 16, 4, I));
    INVALID(extend(I, 2, 3, 3, 9, 16, 4, nullptr));
    UNSUPPORTED(extend(I, 2, 3, 3, 9, 12, 4, I));
    UNSUPPORTED(extend(I, 2, 0x8000000u, 0x8000000u, 9, 16, 4, I));
    UNSUPPORTED(extend(I, 0x8000000u, 3, 3, 9, 16, 4, I));
    UNSUPPORTED(extend(I, 2, 3, 3, 0x80000000u, 16, 4, I));
    UNSUPPORTED(extend(I, 2, 3, 3, 9, 16, 0x7FFFFFFFu, I));
    auto trim = [&](const int32_t* keep, uint32_t seqs, uint32_t cols, uint32_t ld, uint32_t cap,
                    uint32_t page) {
        return w8a8_kv4_trim(keep, I, seqs, I, cols, ld, I, cap, I, page, I, I, st);
    };
    INVALID(trim(nullptr, 2, 3, 3, 9, 16));
    INVALID(trim(I, 2, 3, 1, 9, 16));
    UNSUPPORTED(trim(I, 2, 3, 3, 9, 0));
    UNSUPPORTED(trim(I, 2, 3, 3, 0xFFFFFFFFu, 16));
    UNSUPPORTED(trim(I, 0x100000u, 0x1000u, 0x1000u, 9, 16));

    // ---- page keys ----------------------------------------------------------
    auto bad = [&](auto change, auto use) {
        w8a8_kv4_page_keys k = keys;
        change(k);
        return use(k);
    };
    auto summarize = [&](const w8a8_kv4_page_keys& k) {
        return w8a8_kv4_summarize(&cache, &k, I, 3, 3, I, I, 2, 5, st);
    };
    auto load = [&](const w8a8_kv4_page_keys& k) {
        return w8a8_kv4_page_keys_load(&k, I, 2, static_cast<float*>(P), st);
    };
    auto select = [&](const w8a8_kv4_page_keys& k) {
        return w8a8_kv4_select(P, &k, I, 3, 3, I, 16, I, 2, I, 2, 4, 4 * k.head_dim, nullptr, 0, st);
    };
    auto all = [&](int want, auto change) {
        expect(bad(change, summarize), want, "summarize", __LINE__);
        expect(bad(change, load), want, "load", __LINE__);
        expect(bad(change, select), want, "select", __LINE__);
    };
    all(W8A8_ERROR_INVALID_VALUE, [](w8a8_kv4_page_keys& k) { k.codes = nullptr; });
    all(W8A8_ERROR_INVALID_VALUE, [](w8a8_kv4_page_keys& k) { k.scales = nullptr; });
    all(W8A8_ERROR_INVALID_VALUE, [](w8a8_kv4_page_keys& k) { k.pages = 0; });
    all(W8A8_ERROR_INVALID_VALUE, [](w8a8_kv4_page_keys& k) { k.kv_heads = 70000; });
    all(W8A8_ERROR_NOT_SUPPORTED, [](w8a8_kv4_page_keys& k) { k.head_dim = 32; });
    all(W8A8_ERROR_NOT_SUPPORTED, [](w8a8_kv4_page_keys& k) { k.codes += 4; });
    INVALID(bad([](w8a8_kv4_page_keys& k) { k.pages = 3; }, summarize));
    INVALID(w8a8_kv4_summarize(&cache, nullptr, I, 3, 3, I, I, 2, 5, st));
    INVALID(w8a8_kv4_summarize(nullptr, &keys, I, 3, 3, I, I, 2, 5, st));
    INVALID(w8a8_kv4_summarize(&cache, &keys, nullptr, 3, 3, I, I, 2, 5, st));
    UNSUPPORTED(w8a8_kv4_summarize(&cache, &keys, I, 3, 3, I, I, 0x4000000u, 0x7FFFFFFFu, st));
    DONE(w8a8_kv4_summarize(&cache, &keys, I, 3, 3, I, I, 0, 5, st));
    DONE(w8a8_kv4_summarize(&cache, &keys, I, 3, 3, I, I, 2, 0, st));
    UNSUPPORTED(w8a8_kv4_page_keys_load(&keys, I, 0x8000000u, static_cast<float*>(P), st));
    UNSUPPORTED(w8a8_kv4_page_keys_load(&keys, I, 2, static_cast<float*>(O), st));
    DONE(w8a8_kv4_page_keys_load(&keys, nullptr, 0, nullptr, st));
    auto pick = [&](uint32_t cols, uint32_t keep, uint32_t seqs, uint32_t heads, uint32_t ldq,
                    void* ws, size_t bytes) {
        return w8a8_kv4_select(P, &keys, I, cols, cols, I, 16, I, keep, I, seqs, heads, ldq, ws,
                               bytes, st);
    };
    INVALID(pick(3, 0, 2, 4, 256, nullptr, 0));
    INVALID(pick(3, 2, 2, 3, 256, nullptr, 0));
    INVALID(pick(3, 2, 2, 4, 248, nullptr, 0));
    INVALID(pick(9000, 2, 2, 4, 256, nullptr, 0));
    INVALID(pick(9000, 2, 2, 4, 256, O, 1u << 30));
    INVALID(pick(9000, 2, 2, 4, 256, P, 100));
    UNSUPPORTED(pick(3, 0x7FFFFFFFu, 2, 4, 256, nullptr, 0));
    UNSUPPORTED(pick(3, 2, 0x400000u, 4, 256, nullptr, 0));
    DONE(pick(3, 2, 0, 4, 256, nullptr, 0));

    // ---- attention ------------------------------------------------------------
    auto chunks = [&](const void* q, uint32_t cols, uint32_t seqs, uint32_t tokens, uint32_t heads,
                      uint32_t ldq, float scale, void* ws, size_t bytes) {
        return w8a8_attention_kv4_chunks(q, &cache, I, cols, cols, I, I, P, seqs, tokens, heads, 0,
                                         ldq, ldq, scale, ws, bytes, st);
    };
    INVALID(chunks(nullptr, 9, 2, 5, 4, 256, 1.f, P, 1u << 30));
    INVALID(chunks(P, 9, 2, 5, 3, 256, 1.f, P, 1u << 30));
    INVALID(chunks(P, 9, 2, 5, 4, 248, 1.f, P, 1u << 30));
    INVALID(chunks(P, 9, 2, 5, 4, 256, 0.f, P, 1u << 30));
    INVALID(chunks(P, 9, 2, 5, 4, 256, 1.f, nullptr, 0));
    INVALID(chunks(P, 9, 2, 5, 4, 256, 1.f, O, 1u << 30));
    INVALID(chunks(P, 9, 2, 5, 4, 256, 1.f, P, 1000));
    UNSUPPORTED(chunks(O, 9, 2, 5, 4, 256, 1.f, P, 1u << 30));
    UNSUPPORTED(chunks(P, 9, 2, 5, 4, 260, 1.f, P, 1u << 30));
    UNSUPPORTED(chunks(P, 9, 2, 0x80000000u, 4, 256, 1.f, P, 1u << 30));
    UNSUPPORTED(chunks(P, 0x1000000u, 2, 0x100000u, 4, 256, 1.f, P, 1u << 30));
    DONE(chunks(P, 9, 0, 5, 4, 256, 1.f, nullptr, 0));
    DONE(chunks(P, 9, 2, 0, 4, 256, 1.f, nullptr, 0));
    auto over = [&](const void* q, uint32_t cols, uint32_t seqs, uint32_t heads, void* ws) {
        return w8a8_attention_kv4_selected(q, &cache, I, cols, I, P, seqs, heads, 256, 256, 1.f, ws,
                                           0, st);
    };
    INVALID(over(nullptr, 4, 2, 4, nullptr));
    INVALID(over(P, 4, 2, 3, nullptr));
    INVALID(over(P, 4, 2, 4, O));
    UNSUPPORTED(over(O, 4, 2, 4, nullptr));
    UNSUPPORTED(over(P, 0x4000000u, 2, 4, nullptr));
    DONE(over(P, 4, 0, 4, nullptr));

    std::printf("OK %d\n", g_calls);
    return 0;
}
