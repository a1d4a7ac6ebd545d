// kv4.hip -- the paged cache of 4-bit keys and values for gfx950: quantizing
// rows into it, reading rows back, and the attention of single tokens over it.
#include "w8a8_device.hpp"
#include "w8a8_internal.hpp"

#include <algorithm>

namespace w8a8 {
namespace {

constexpr int kRowThreads = 256;

struct CacheView {
    uint8_t*  codes[2];  // keys, values
    uint32_t* scales[2]; // (scale, offset) fp16 pairs
    uint32_t  slots;     // pages * page_size
    uint32_t  page_shift, page_size, kv_heads;
};

CacheView view(const w8a8_kv4_cache& c)
{
    return {{c.k_codes, c.v_codes},
            {static_cast<uint32_t*>(c.k_scales), static_cast<uint32_t*>(c.v_scales)},
            c.pages * c.page_size,
            (uint32_t)__builtin_ctz(c.page_size),
            c.page_size,
            c.kv_heads};
}

// Row number of (page, head, place) in the codes and scales.
__device__ __forceinline__ size_t cache_row(const CacheView& c, uint32_t page, uint32_t head,
                                            uint32_t place)
{
    return ((size_t)page * c.kv_heads + head) * c.page_size + place;
}

// Byte of the dword that holds channels 8 * chunk .. 8 * chunk + 7 of a row.
template <int D>
__device__ __forceinline__ uint32_t code_byte(bool keys, uint32_t chunk)
{
    return keys ? (chunk % 4) * (D / 8) + (chunk / 4) * 4 : chunk * 4;
}

// Where thread `at` of the store and load kernels works: 8 channels (16 bytes
// of fp16) of one token's key or value head.  Neighbouring threads take
// neighbouring chunks, so the fp16 side moves whole lines.
template <int D>
struct RowChunk {
    uint32_t chunk, head, side;
    uint64_t token;
    bool     live;
    size_t   row;

    __device__ RowChunk(const CacheView& c, const Kv4Rows& r, uint64_t at)
    {
        chunk = at % (D / 8);
        at /= D / 8;
        head = at % c.kv_heads;
        at /= c.kv_heads;
        side  = at % 2;
        token = at / 2;
        live  = token < r.tokens;
        row   = 0;
        if(live) {
            const int32_t slot = r.slots[token];
            live               = slot >= 0 && (uint32_t)slot < c.slots;
            if(live)
                row = cache_row(c, (uint32_t)slot >> c.page_shift, head,
                                (uint32_t)slot & (c.page_size - 1));
        }
    }
};

// One step of a reduction over the G / 8 lanes of a group.
template <int G, class Op>
__device__ __forceinline__ float group_reduce(float v, Op op)
{
    v = op(v, dpp_mov<kDppQuadXor1>(v));
    v = op(v, dpp_mov<kDppQuadXor2>(v));
    if constexpr(G >= 64) v = op(v, dpp_mov<kDppRowHalfMirror>(v));
    if constexpr(G >= 128) v = op(v, dpp_mov<kDppRowMirror>(v));
    return v;
}

// Quantizes 8 channels a thread; the G / 8 threads of a group share its minimum
// and maximum by DPP.  Memory bound: 16 bytes read and 4 (+ 4 / 4 of scales)
// written per thread.
template <int D, int G>
__global__ void __launch_bounds__(kRowThreads)
    kv4_store_kernel(CacheView c, Kv4Rows r, const uint16_t* __restrict__ k,
                     const uint16_t* __restrict__ v)
{
    const RowChunk<D> t(c, r, (uint64_t)blockIdx.x * kRowThreads + threadIdx.x);
    // groups are whole within a token, so the lanes of a group are live together
    float x[8];
    float low = INFINITY, high = -INFINITY, bad = 0.f;
    v4i   raw = {};
    if(t.live)
        raw = *reinterpret_cast<const v4i*>((t.side ? v + t.token * r.ldv : k + t.token * r.ldk)
                                            + t.head * D + t.chunk * 8);
#pragma unroll
    for(int i = 0; i < 8; ++i) {
        x[i] = half_bits_to_float((uint32_t)raw[i / 2] >> (16 * (i % 2)));
        low  = fminf(low, x[i]);
        high = fmaxf(high, x[i]);
        bad += x[i] * 0.f; // NaN where x is an infinity or NaN
    }
    low  = group_reduce<G>(low, [](float a, float b) { return fminf(a, b); });
    high = group_reduce<G>(high, [](float a, float b) { return fmaxf(a, b); });
    bad  = group_reduce<G>(bad, [](float a, float b) { return a + b; });
    if(!t.live) return;
    uint32_t     s16 = float_to_half_bits((high - low) / 15.f);
    const float  s   = half_bits_to_float(s16);
    uint32_t     c16 = float_to_half_bits_2step(fmaf(8.f, s, low));
    const float  mid = half_bits_to_float(c16);
    const bool   ok  = bad == 0.f;
    if(!ok) s16 = c16 = 0x7E00u;
    uint32_t codes = 0;
#pragma unroll
    for(int i = 0; i < 8; ++i) {
        const float n = s > 0.f && ok
                            ? fminf(fmaxf(__builtin_rintf((x[i] - mid) / s) + 8.f, 0.f), 15.f)
                            : 8.f;
        codes |= (uint32_t)n << (4 * i);
    }
    *reinterpret_cast<uint32_t*>(c.codes[t.side] + t.row * (D / 2)
                                 + code_byte<D>(t.side == 0, t.chunk))
        = codes;
    if(t.chunk % (G / 8) == 0)
        c.scales[t.side][t.row * (D / G) + t.chunk / (G / 8)] = s16 | (c16 << 16);
}

template <int D, int G>
__global__ void __launch_bounds__(kRowThreads)
    kv4_load_kernel(CacheView c, Kv4Rows r, uint16_t* __restrict__ k, uint16_t* __restrict__ v)
{
    const RowChunk<D> t(c, r, (uint64_t)blockIdx.x * kRowThreads + threadIdx.x);
    if(!t.live) return;
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(
        c.codes[t.side] + t.row * (D / 2) + code_byte<D>(t.side == 0, t.chunk));
    const uint32_t sc  = c.scales[t.side][t.row * (D / G) + t.chunk / (G / 8)];
    const float    s   = half_bits_to_float(sc & 0xFFFFu);
    const float    mid = half_bits_to_float(sc >> 16);
    v4i            out;
#pragma unroll
    for(int i = 0; i < 4; ++i) {
        const float a = fmaf(s, (float)((codes >> (8 * i)) & 15u) - 8.f, mid);
        const float b = fmaf(s, (float)((codes >> (8 * i + 4)) & 15u) - 8.f, mid);
        out[i]        = (int)float2_to_half2_bits_2step(a, b);
    }
    *reinterpret_cast<v4i*>((t.side ? v + t.token * r.ldv : k + t.token * r.ldk) + t.head * D
                            + t.chunk * 8)
        = out;
}

// The instantiation for a cache's head width and group.
template <class F>
void with_widths(const w8a8_kv4_cache& c, F f)
{
    using std::integral_constant;
    if(c.head_dim == 64) {
        if(c.group == 32)
            f(integral_constant<int, 64>(), integral_constant<int, 32>());
        else
            f(integral_constant<int, 64>(), integral_constant<int, 64>());
    } else {
        if(c.group == 32)
            f(integral_constant<int, 128>(), integral_constant<int, 32>());
        else if(c.group == 64)
            f(integral_constant<int, 128>(), integral_constant<int, 64>());
        else
            f(integral_constant<int, 128>(), integral_constant<int, 128>());
    }
}

uint32_t row_blocks(const w8a8_kv4_cache& c, const Kv4Rows& r)
{
    const uint64_t threads = (uint64_t)r.tokens * 2 * c.kv_heads * (c.head_dim / 8);
    return (uint32_t)((threads + kRowThreads - 1) / kRowThreads);
}

// One wave per (sequence, head): lanes over the channels, one token after the
// other with a running maximum and sum.
template <int D, int G>
__global__ void __launch_bounds__(kWave)
    attention_kv4_kernel(CacheView c, AttentionKv4Args a, uint32_t pages)
{
    constexpr int  kC   = D / kWave; // channels per lane: 2 lane, 2 lane + 1, or lane
    const uint32_t head = blockIdx.x, seq = blockIdx.y, lane = threadIdx.x;
    const uint32_t kvh  = head / (a.heads / c.kv_heads);
    const uint32_t ch0  = lane * kC;
    float          q[kC], o[kC];
#pragma unroll
    for(int i = 0; i < kC; ++i) {
        q[i] = half_bits_to_float(a.q[(size_t)seq * a.ldq + head * D + ch0 + i]) * a.scale;
        o[i] = 0.f;
    }
    const int64_t most = (int64_t)a.table_cols * c.page_size;
    const int64_t len  = max((int64_t)0, min((int64_t)a.lens[seq], most));
    float         m = -INFINITY, l = 0.f;
    for(int64_t t = 0; t < len; ++t) {
        const int32_t page = a.table[(size_t)seq * a.table_ld + (t >> c.page_shift)];
        if(page < 0 || (uint32_t)page >= pages) continue;
        const size_t row = cache_row(c, page, kvh, t & (c.page_size - 1));
        float        v[2][kC];
#pragma unroll
        for(int side = 0; side < 2; ++side)
#pragma unroll
            for(int i = 0; i < kC; ++i) {
                const uint32_t ch = ch0 + i;
                const uint32_t b  = c.codes[side][row * (D / 2) + code_byte<D>(side == 0, ch / 8)
                                                 + ch % 8 / 2];
                const uint32_t sc = c.scales[side][row * (D / G) + ch / G];
                v[side][i] = fmaf(half_bits_to_float(sc & 0xFFFFu),
                                  (float)((b >> (4 * (ch % 2))) & 15u) - 8.f,
                                  half_bits_to_float(sc >> 16));
            }
        float dot = 0.f;
#pragma unroll
        for(int i = 0; i < kC; ++i) dot = fmaf(q[i], v[0][i], dot);
        const float s  = wave_sum(dot);
        const float mn = fmaxf(m, s);
        const float al = m == mn ? 1.f : __expf(m - mn), p = s == mn ? 1.f : __expf(s - mn);
        m              = mn;
        l              = l * al + p;
#pragma unroll
        for(int i = 0; i < kC; ++i) o[i] = o[i] * al + p * v[1][i];
    }
#pragma unroll
    for(int i = 0; i < kC; ++i)
        a.out[(size_t)seq * a.ldo + head * D + ch0 + i] = float_to_half_bits(l != 0.f ? o[i] / l : 0.f);
}

} // namespace

hipError_t launch_kv4_store(const w8a8_kv4_cache& c, const Kv4Rows& r, const uint16_t* k,
                            const uint16_t* v, hipStream_t stream)
{
    with_widths(c, [&](auto d, auto g) {
        kv4_store_kernel<d(), g()><<<row_blocks(c, r), kRowThreads, 0, stream>>>(view(c), r, k, v);
    });
    return hipGetLastError();
}

hipError_t launch_kv4_load(const w8a8_kv4_cache& c, const Kv4Rows& r, uint16_t* k, uint16_t* v,
                           hipStream_t stream)
{
    with_widths(c, [&](auto d, auto g) {
        kv4_load_kernel<d(), g()><<<row_blocks(c, r), kRowThreads, 0, stream>>>(view(c), r, k, v);
    });
    return hipGetLastError();
}

size_t attention_kv4_workspace_bytes(uint32_t seqs, uint32_t heads, uint32_t kv_heads, uint32_t dim,
                                     uint32_t max_len)
{
    return 0;
}

hipError_t launch_attention_kv4(const w8a8_kv4_cache& c, const AttentionKv4Args& a,
                                hipStream_t stream)
{
    with_widths(c, [&](auto d, auto g) {
        attention_kv4_kernel<d(), g()>
            <<<dim3(a.heads, a.seqs), kWave, 0, stream>>>(view(c), a, c.pages);
    });
    return hipGetLastError();
}

} // namespace w8a8
