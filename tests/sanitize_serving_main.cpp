// Driver of the host side of attention, the 4-bit cache and the expert layer of few tokens
// for the sanitizer build of test_sanitizers_serving_cpu.py: every entry point with
// arguments its checks reject, its size queries over a range of shapes, and the calls that
// have nothing to do.  Nothing here reaches a kernel launch, and no pointer below is
// dereferenced but the cache descriptor's.  Prints "OK <calls>" on success.
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
    void*          P = reinterpret_cast<void*>(0x100000);
    void*          O = reinterpret_cast<void*>(0x100008); // off the 16-byte alignment
    const int32_t* I = static_cast<const int32_t*>(P);
    const int8_t*  W = static_cast<const int8_t*>(P);
    const float*   F = static_cast<const float*>(P);
    hipStream_t    st = nullptr;

    // ---- size queries -------------------------------------------------------
    size_t sink = 0;
    for(uint32_t t : {1u, 2u, 16u})
        for(uint32_t k : {1u, 6u, 32u})
            for(uint32_t h : {16u, 1040u, 7168u, 32768u})
                for(uint32_t i : {16u, 1408u, 32768u})
                    sink += w8a8_moe_ffn_decode_workspace_size(t, k, h, i);
    for(uint32_t s : {0u, 1u, 48u, 65536u})
        for(uint32_t h : {0u, 1u, 8u, 64u, 65535u})
            for(uint32_t kh : {0u, 1u, 3u, 8u})
                for(uint32_t d : {64u, 128u})
                    for(uint32_t len : {0u, 1u, 64u, 65u, 131072u, 0x7FFFFFFFu})
                        sink += w8a8_attention_kv4_workspace_size(s, h, kh, d, len);
    if(sink == 0) return 1;

    // ---- attention of prompts ----------------------------------------------------
    auto att = [&](void* q, void* k, void* v, void* o, const int32_t* starts, uint32_t seqs,
                   uint32_t tokens, uint32_t heads, uint32_t kvh, uint32_t dim, uint32_t ldq,
                   uint32_t ldk, uint32_t ldv, uint32_t ldo, float scale) {
        return w8a8_attention(q, k, v, o, starts, seqs, tokens, heads, kvh, dim, ldq, ldk, ldv, ldo,
                              scale, st);
    };
    INVALID(att(nullptr, P, P, P, I, 1, 8, 4, 2, 64, 256, 128, 128, 256, 1.f));
    INVALID(att(P, P, P, P, nullptr, 1, 8, 4, 2, 64, 256, 128, 128, 256, 1.f));
    INVALID(att(P, P, P, P, I, 1, 8, 4, 3, 64, 256, 192, 192, 256, 1.f));
    INVALID(att(P, P, P, P, I, 1, 8, 0, 1, 64, 256, 192, 192, 256, 1.f));
    UNSUPPORTED(att(P, P, P, P, I, 1, 8, 4, 2, 96, 384, 192, 192, 384, 1.f));
    INVALID(att(P, P, P, P, I, 1, 8, 4, 2, 64, 248, 128, 128, 256, 1.f));
    INVALID(att(P, P, P, P, I, 1, 8, 4, 2, 64, 256, 120, 128, 256, 1.f));
    UNSUPPORTED(att(P, P, P, P, I, 1, 8, 4, 2, 64, 260, 128, 128, 256, 1.f));
    UNSUPPORTED(att(O, P, P, P, I, 1, 8, 4, 2, 64, 256, 128, 128, 256, 1.f));
    UNSUPPORTED(att(P, P, P, P, I, 0x400000u, 8, 4, 2, 64, 256, 128, 128, 256, 1.f)); // threads
    for(float s : {0.f, -1.f, INFINITY, NAN})
        INVALID(att(P, P, P, P, I, 1, 8, 4, 2, 64, 256, 128, 128, 256, s));
    DONE(att(P, P, P, P, I, 0, 8, 4, 2, 64, 256, 128, 128, 256, 1.f));
    DONE(att(P, P, P, P, I, 1, 0, 4, 2, 64, 256, 128, 128, 256, 1.f));

    // ---- the cache ------------------------------------------------------------------
    uint8_t*             B    = static_cast<uint8_t*>(P);
    const w8a8_kv4_cache good = {B, B, P, P, 4, 32, 2, 64, 32};
    auto bad = [&](auto change, auto use) {
        w8a8_kv4_cache c = good;
        change(c);
        return use(c);
    };
    auto store = [&](const w8a8_kv4_cache& c) {
        return w8a8_kv4_store(P, P, I, 3, 128, 128, &c, st);
    };
    auto load = [&](const w8a8_kv4_cache& c) { return w8a8_kv4_load(P, P, I, 3, 128, 128, &c, st); };
    auto over = [&](const w8a8_kv4_cache& c) {
        return w8a8_attention_kv4(P, &c, I, 4, 4, I, P, 2, 4, 4 * c.head_dim, 4 * c.head_dim, 1.f,
                                  nullptr, 0, st);
    };
    auto all = [&](int want, auto change) {
        expect(bad(change, store), want, "store", __LINE__);
        expect(bad(change, load), want, "load", __LINE__);
        expect(bad(change, over), want, "attention", __LINE__);
    };
    all(W8A8_ERROR_INVALID_VALUE, [](w8a8_kv4_cache& c) { c.k_codes = nullptr; });
    all(W8A8_ERROR_INVALID_VALUE, [](w8a8_kv4_cache& c) { c.v_scales = nullptr; });
    all(W8A8_ERROR_INVALID_VALUE, [](w8a8_kv4_cache& c) { c.pages = 0; });
    all(W8A8_ERROR_INVALID_VALUE, [](w8a8_kv4_cache& c) { c.kv_heads = 0; });
    all(W8A8_ERROR_NOT_SUPPORTED, [](w8a8_kv4_cache& c) { c.head_dim = 80; });
    all(W8A8_ERROR_NOT_SUPPORTED, [](w8a8_kv4_cache& c) { c.group = 128; });
    all(W8A8_ERROR_NOT_SUPPORTED, [](w8a8_kv4_cache& c) { c.group = 16; });
    all(W8A8_ERROR_NOT_SUPPORTED, [](w8a8_kv4_cache& c) { c.page_size = 24; });
    all(W8A8_ERROR_NOT_SUPPORTED, [](w8a8_kv4_cache& c) { c.page_size = 2048; });
    all(W8A8_ERROR_NOT_SUPPORTED, [](w8a8_kv4_cache& c) { c.pages = 0xFFFFFFFFu; });
    all(W8A8_ERROR_NOT_SUPPORTED, [](w8a8_kv4_cache& c) { c.v_codes += 8; });
    INVALID(w8a8_kv4_store(P, P, I, 3, 128, 128, nullptr, st));
    INVALID(w8a8_kv4_store(P, nullptr, I, 3, 128, 128, &good, st));
    INVALID(w8a8_kv4_store(P, P, nullptr, 3, 128, 128, &good, st));
    INVALID(w8a8_kv4_store(P, P, I, 3, 120, 128, &good, st));
    UNSUPPORTED(w8a8_kv4_store(P, P, I, 3, 132, 128, &good, st));
    UNSUPPORTED(w8a8_kv4_store(O, P, I, 3, 128, 128, &good, st));
    UNSUPPORTED(w8a8_kv4_load(P, O, I, 3, 128, 128, &good, st));
    UNSUPPORTED(w8a8_kv4_store(P, P, I, 0x10000000u, 128, 128, &good, st)); // threads
    DONE(w8a8_kv4_store(nullptr, nullptr, nullptr, 0, 0, 0, &good, st));
    DONE(w8a8_kv4_load(nullptr, nullptr, nullptr, 0, 0, 0, &good, st));

    // ---- attention over it ----------------------------------------------------------
    auto dec = [&](const void* q, uint32_t cols, uint32_t ld, uint32_t seqs, uint32_t heads,
                   uint32_t ldq, float scale, void* ws) {
        return w8a8_attention_kv4(q, &good, I, cols, ld, I, P, seqs, heads, ldq, ldq, scale, ws, 0,
                                  st);
    };
    INVALID(dec(nullptr, 4, 4, 2, 4, 256, 1.f, nullptr));
    INVALID(dec(P, 4, 3, 2, 4, 256, 1.f, nullptr));
    INVALID(dec(P, 4, 4, 2, 3, 256, 1.f, nullptr));
    INVALID(dec(P, 4, 4, 2, 4, 248, 1.f, nullptr));
    INVALID(dec(P, 4, 4, 2, 4, 256, 0.f, nullptr));
    INVALID(dec(P, 4, 4, 2, 4, 256, 1.f, O));
    UNSUPPORTED(dec(O, 4, 4, 2, 4, 256, 1.f, nullptr));
    UNSUPPORTED(dec(P, 4, 4, 2, 4, 260, 1.f, nullptr));
    UNSUPPORTED(dec(P, 0x4000000u, 0x4000000u, 2, 4, 256, 1.f, nullptr)); // 2^31 tokens
    UNSUPPORTED(dec(P, 4, 4, 0x1000000u, 4, 256, 1.f, nullptr));
    UNSUPPORTED(dec(P, 0x100000u, 0x100000u, 0x10000u, 4, 256, 1.f, nullptr)); // chunks
    DONE(dec(P, 4, 4, 0, 4, 256, 1.f, nullptr));

    // ---- the expert layer -----------------------------------------------------------
    struct Moe {
        const void* x     = reinterpret_cast<void*>(0x100000);
        uint32_t    tokens = 2, hidden = 64, inter = 32, experts = 4, topk = 2, ldx = 64, ldo = 64;
        float       qmax   = 127.f;
        void*       ws     = reinterpret_cast<void*>(0x100000);
        size_t      bytes  = 1u << 30;
    };
    auto moe = [&](auto change) {
        Moe m;
        change(m);
        return w8a8_moe_ffn_decode(m.x, P, 1, F, W, F, F, W, F, P, m.tokens, m.hidden, m.inter,
                                   m.experts, m.topk, m.qmax, m.ldx, m.ldo, m.ws, m.bytes, st);
    };
    INVALID(moe([](Moe& m) { m.x = nullptr; }));
    INVALID(moe([](Moe& m) { m.ws = nullptr; }));
    INVALID(moe([](Moe& m) { m.hidden = 0; }));
    INVALID(moe([](Moe& m) { m.topk = 5; }));
    INVALID(moe([](Moe& m) { m.qmax = 128.f; }));
    INVALID(moe([](Moe& m) { m.ldx = 56; }));
    INVALID(moe([](Moe& m) { m.ws = static_cast<char*>(m.ws) + 64; }));
    INVALID(moe([](Moe& m) { m.bytes = 16; }));
    UNSUPPORTED(moe([](Moe& m) { m.tokens = 17; }));
    UNSUPPORTED(moe([](Moe& m) { m.tokens = 16, m.hidden = m.ldx = m.ldo = 7184; }));
    UNSUPPORTED(moe([](Moe& m) { m.experts = 4097; }));
    UNSUPPORTED(moe([](Moe& m) { m.experts = 64, m.topk = 33; }));
    UNSUPPORTED(moe([](Moe& m) { m.hidden = m.ldx = m.ldo = 72; }));
    UNSUPPORTED(moe([](Moe& m) { m.inter = 40; }));
    UNSUPPORTED(moe([](Moe& m) { m.inter = 32784; }));
    UNSUPPORTED(moe([](Moe& m) { m.ldx = 68; }));
    UNSUPPORTED(moe([](Moe& m) { m.x = static_cast<const char*>(m.x) + 8; }));
    DONE(moe([](Moe& m) { m.tokens = 0; }));

    std::printf("OK %d\n", g_calls);
    return 0;
}
