// kv4.hip -- the paged cache of 4-bit keys and values for gfx950: quantizing
// rows into it, reading rows back, and the attention of single tokens over it.
#include "w8a8_device.hpp"
#include "w8a8_internal.hpp"

#include <algorithm>

namespace w8a8 {
namespace {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

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

// How the store and load kernels share out their work: a thread takes 8 channels (16
// bytes of fp16) of one token and head, of its keys and of its values.  Neighbouring
// threads take neighbouring channels, so the fp16 side moves whole lines; a block has
// some whole tokens, and the blocks of one XCD have neighbouring ones, whose rows share
// lines of the cache (heads, not tokens, lie a page apart there).
// (Keys and values by threads of their own, each finding its place by two divisions of
// 64 bits, took 18.9 us to store and 12.8 to load 8192 tokens of 8 heads of 128; this
// takes 11.3 and 8.7, and with two or four chunks a thread 13.3 and 15.6 to store.)
struct RowPlan {
    uint32_t blocks;    // a multiple of 8
    uint32_t tokens;    // a block's
    uint32_t per_token; // chunks of a token's keys or values
    uint32_t inverse;   // ceil(2^32 / per_token) where a block has several tokens, else 0
};

// The block's first token, `tokens` where it has none: an XCD (block number modulo 8)
// has a contiguous run.
__device__ __forceinline__ uint32_t first_token(const RowPlan& p, uint32_t tokens)
{
    const uint32_t at = blockIdx.x % 8 * (p.blocks / 8) + blockIdx.x / 8;
    return (uint32_t)min((uint64_t)at * p.tokens, (uint64_t)tokens);
}

// Where a block's i-th chunk is.
template <int D>
struct RowChunk {
    uint32_t chunk, head, token;
    size_t   row; // in the cache

    __device__ RowChunk(const RowPlan& p, uint32_t token0, uint32_t i)
    {
        // exact: i * (inverse * per_token - 2^32) < 2^32, as a block has few chunks
        // where inverse is not 0
        const uint32_t t  = __umulhi(i, p.inverse);
        const uint32_t at = i - t * p.per_token;
        chunk             = at % (D / 8);
        head              = at / (D / 8);
        token             = token0 + t;
    }

    // its row; false where the slot lies outside the cache
    __device__ bool place(const CacheView& c, int32_t slot)
    {
        if(slot < 0 || (uint32_t)slot >= c.slots) return false;
        const uint32_t at = (uint32_t)slot;
        row = cache_row(c, at >> c.page_shift, head, at & (c.page_size - 1));
        return true;
    }
};

// One step of a reduction over the G / 8 lanes of a group.
template <int G, class T, class Op>
__device__ __forceinline__ T group_reduce(T v, Op op)
{
    const auto step = [&](auto dpp) {
        const float o = dpp_mov<decltype(dpp)::value>(__builtin_bit_cast(float, v));
        v             = op(v, __builtin_bit_cast(T, o));
    };
    step(std::integral_constant<int, kDppQuadXor1>());
    step(std::integral_constant<int, kDppQuadXor2>());
    if constexpr(G >= 64) step(std::integral_constant<int, kDppRowHalfMirror>());
    if constexpr(G >= 128) step(std::integral_constant<int, kDppRowMirror>());
    return v;
}

// a / b rounded once, y = 1 / b rounded once (Markstein's theorem: the product and one
// correction by the exact remainder), for quotients far from the ends of fp32's range.
__device__ __forceinline__ float quotient(float a, float b, float y)
{
    const float q = a * y;
    return fmaf(fmaf(-q, b, a), y, q);
}

// Two fp32 results as packed fp16, those past its range as its ends: the last code of a
// group that reaches 65504 may stand for a little more, its step being rounded (0 .. 65504
// has steps of 4368 and ends at 65520, which would be an infinity).  NaN stays NaN.
__device__ __forceinline__ uint32_t finite_halves(float a, float b)
{
    const v2h most = {(_Float16)65504.f, (_Float16)65504.f};
    const v2h h    = __builtin_bit_cast(v2h, float2_to_half2_bits_2step(a, b));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_minimum(
                                            __builtin_elementwise_maximum(h, -most), most));
}

// The 8 codes of a thread's channels and its group's (scale, offset).
template <int G>
__device__ __forceinline__ v2i quantized(v4i raw)
{
    // the group's extremes, two channels a register, NaN if one is
    const auto x = __builtin_bit_cast(v8h, raw);
    v2h        low = {x[0], x[1]}, high = low;
#pragma unroll
    for(int i = 2; i < 8; i += 2) {
        const v2h h = {x[i], x[i + 1]};
        low         = __builtin_elementwise_minimum(low, h);
        high        = __builtin_elementwise_maximum(high, h);
    }
    low  = group_reduce<G>(low, [](v2h a, v2h b) { return __builtin_elementwise_minimum(a, b); });
    high = group_reduce<G>(high, [](v2h a, v2h b) { return __builtin_elementwise_maximum(a, b); });
    const float lo = (float)__builtin_elementwise_minimum(low[0], low[1]);
    const float hi = (float)__builtin_elementwise_maximum(high[0], high[1]);

    uint32_t    s16 = float_to_half_bits(quotient(hi - lo, 15.f, 1.f / 15.f));
    const float s   = half_bits_to_float(s16);
    uint32_t    c16 = float_to_half_bits_2step(fmaf(8.f, s, lo));
    const float mid = half_bits_to_float(c16);
    const bool  ok  = (hi - lo) * 0.f == 0.f; // no infinity and no NaN
    if(!ok) s16 = c16 = 0x7E00u;
    // A code is clamp(rint((x - mid) / s), -8, 7) + 8, and 8 where s is 0 or not finite
    // (then y = 0).  Adding kRound rounds to an integer, which the sum's low bits
    // hold; its other bits times the places' weights add up to kRest.
    const float        y      = s > 0.f && ok ? 1.f / s : 0.f;
    const float        from   = ok ? mid : 0.f;
    constexpr float    kRound = 12582912.f + 8.f; // 1.5 2^23: units of 1
    constexpr uint32_t kRest  = 0x4B400000u * 0x11111111u;
    uint32_t           codes  = 0u - kRest;
#pragma unroll
    for(int i = 0; i < 8; ++i) {
        const float q = __builtin_amdgcn_fmed3f(quotient((float)x[i] - from, s, y), -8.f, 7.f);
        codes += __float_as_uint(q + kRound) << (4 * i);
    }
    return v2i{(int)(ok ? codes : 0x88888888u), (int)(s16 | (c16 << 16))};
}

// Quantizes rows.  Bound by memory: 16 bytes read and 4 (and 4 of scales a group)
// written per 8 channels.
template <int D, int G>
__global__ void __launch_bounds__(kRowThreads)
    kv4_store_kernel(CacheView c, Kv4Rows r, RowPlan p, const uint16_t* __restrict__ k,
                     const uint16_t* __restrict__ v)
{
    const uint32_t token0 = first_token(p, r.tokens);
    const uint32_t count  = min(p.tokens, r.tokens - token0) * p.per_token;
    for(uint32_t i = threadIdx.x; i < count; i += kRowThreads) {
        RowChunk<D>    t(p, token0, i);
        const uint32_t at     = t.head * D + t.chunk * 8;
        const int32_t  slot   = r.slots[t.token];
        const v4i      raw[2] = {*reinterpret_cast<const v4i*>(k + (size_t)t.token * r.ldk + at),
                                 *reinterpret_cast<const v4i*>(v + (size_t)t.token * r.ldv + at)};
        // groups are whole within a token: their lanes go on together
        if(!t.place(c, slot)) continue;
#pragma unroll
        for(int side = 0; side < 2; ++side) {
            const v2i q = quantized<G>(raw[side]);
            *reinterpret_cast<int32_t*>(c.codes[side] + t.row * (D / 2)
                                        + code_byte<D>(side == 0, t.chunk))
                = q[0];
            if(t.chunk % (G / 8) == 0)
                c.scales[side][t.row * (D / G) + t.chunk / (G / 8)] = (uint32_t)q[1];
        }
    }
}

template <int D, int G>
__global__ void __launch_bounds__(kRowThreads)
    kv4_load_kernel(CacheView c, Kv4Rows r, RowPlan p, uint16_t* __restrict__ k,
                    uint16_t* __restrict__ v)
{
    const uint32_t token0 = first_token(p, r.tokens);
    const uint32_t count  = min(p.tokens, r.tokens - token0) * p.per_token;
    for(uint32_t i = threadIdx.x; i < count; i += kRowThreads) {
        RowChunk<D> t(p, token0, i);
        if(!t.place(c, r.slots[t.token])) continue;
        uint32_t codes[2], scales[2];
#pragma unroll
        for(int side = 0; side < 2; ++side) {
            codes[side] = *reinterpret_cast<const uint32_t*>(
                c.codes[side] + t.row * (D / 2) + code_byte<D>(side == 0, t.chunk));
            scales[side] = c.scales[side][t.row * (D / G) + t.chunk / (G / 8)];
        }
#pragma unroll
        for(int side = 0; side < 2; ++side) {
            const float s   = half_bits_to_float(scales[side] & 0xFFFFu);
            const float mid = half_bits_to_float(scales[side] >> 16);
            v4i         out;
#pragma unroll
            for(int j = 0; j < 4; ++j) {
                const uint32_t w = codes[side] >> (8 * j);
                const float    a = fmaf(s, (float)(w & 15u) - 8.f, mid);
                const float    b = fmaf(s, (float)(w >> 4 & 15u) - 8.f, mid);
                out[j]           = (int)finite_halves(a, b);
            }
            uint16_t* to = side ? v + (size_t)t.token * r.ldv : k + (size_t)t.token * r.ldk;
            *reinterpret_cast<v4i*>(to + t.head * D + t.chunk * 8) = out;
        }
    }
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

// As many tokens a block as one round of its threads takes, and one where that is less.
RowPlan row_plan(const w8a8_kv4_cache& c, const Kv4Rows& r)
{
    const uint32_t per_token = c.kv_heads * (c.head_dim / 8);
    const uint32_t tokens    = std::max(1u, kRowThreads / per_token);
    const uint32_t inverse
        = tokens > 1 ? (uint32_t)(((1ull << 32) + per_token - 1) / per_token) : 0;
    const uint32_t blocks = (uint32_t)(((uint64_t)r.tokens + tokens - 1) / tokens);
    return {(blocks + 7) / 8 * 8, tokens, per_token, inverse};
}

// ---------------------------------------------------------------------------
// Attention of single tokens over the cache.
//
// The chunks of 64 tokens of all (sequence, key head) units lie in one line, which is
// cut into as many equal runs as there are waves; every wave works through its run by
// itself, its next chunk on the way while it computes.  A unit inside one run is
// written out; of one cut by runs each wave leaves a partial (its sum of p v, maximum
// and sum of p), and a second launch joins them in order.  So any mix of lengths
// keeps the chip evenly busy.  131072 tokens, 32 / 8 heads of 128, 168 MB: 39 us and 5 of
// the join, 4.3 TB/s, 5.0 behind the 5.5 us of start (lengths, page numbers, then codes);
// 48 sequences of 249 MB in all 62 and 5, 4.0 TB/s.  Bound by a wave's chain from chunk to
// chunk and its 690 vector instructions: the page number of the chunk after next is waited
// for where it is loaded, ahead of the next chunk's loads, and the queue is empty again at
// the loop's end.  (Blocks that owned a piece of one sequence spent 10 of their 18 us on
// starting, the first load and merging: 16 x 8192 tokens 42 us.)
// Both products run on v_mfma_f32_16x16x32_f16 with the query heads as columns:
//   S^T = K q^T    srcA rows = tokens.  A lane takes 16 (8) bytes of one token's
//                  codes; dword j is its operand of step j, channels 32 j + 8 kg +
//                  0..7 (kg = lane / 16), which is the cache's order of keys.
//   O^T = V^T P^T  srcA rows = channels: ds_read_b64_tr_b4 turns 16 tokens x 16
//                  channels of row-major codes in LDS into 16 tokens of one channel
//                  per lane.  The tokens a lane's S^T registers hold (4 kg .. 4 kg + 3
//                  of each 16) are the ones its P^T operand needs: nothing moves
//                  between lanes.
// Codes are not scaled into fp16 values: a code n enters as 1 + n / 16, two bit
// operations a pair and exact, and scales and offsets are applied where they are
// per-lane fp32 factors,
//   q . k    = sum over groups of 16 s (sum_c q_c (x_c - 1.5)) + o (sum_c q_c)
//   (p v)_c  = 16 (sum_t (p s)_t x_c,t - 1.5 sum_t (p s)_t) + sum_t (p o)_t
// (the -1.5 makes x the centred code; in O^T with
// the sum over the tokens of the rounded p s, from a matrix product with ones, so
// that rounding p s to fp16, the only rounding below fp32, acts on the centred
// code).  p s is brought to fp16's range by a power of two that follows the scales: one a
// chunk and key head, taken from its largest scale s, which then lies between 1 and 64.  A
// p s below 2^-14 has fewer than fp16's 11 bits and one below 2^-25 none, so the centred
// codes of a group whose scales are a small part of the largest lose precision (their
// offsets, in fp32, do not).  The two held sums cancel 1.5 of each code in fp32: some 2^-20
// of the largest scale is left where a result is far smaller than that.  A power for each group would take its own maximum, rescaling
// and product a group in a loop that is bound by such instructions.
//
// With few query heads per key head most of the 16 columns would hold nothing, and
// the work on scores, which is per column, would be done for nothing.  So C = 4 or 2
// copies of 4 or 8 heads fill them, copy (class) a for every C-th of the chunk's four
// 16-token tiles: the tile's product takes a q^T whose other classes are zero, and the
// products of C tiles add up in one accumulator.  A column is then a partial of its
// own, with its own maximum, sum and part of the result, merged at the unit's end.
// ---------------------------------------------------------------------------
typedef float    v2f __attribute__((ext_vector_type(2)));

typedef __attribute__((address_space(3))) v2i      lds_v2i_t;
typedef __attribute__((address_space(3))) v4i      lds_v4i_t;
typedef __attribute__((address_space(3))) uint32_t lds_u32_t;

constexpr int      kAttWaves   = 4;
constexpr int      kAttThreads = kAttWaves * kWave;
constexpr uint32_t kAttBlocks  = 512; // two a CU, all resident: 2 waves a SIMD by registers
constexpr int      kChunk      = 64;  // tokens a wave takes at a time
constexpr int      kCols       = 16;  // columns of a product: classes x query heads

// The 8 codes of a dword as fp16 1 + n / 16, in the order 0 4 1 5 2 6 3 7: a shift
// and a v_and_or_b32 a pair.  The constants come in registers, which that
// instruction needs on gfx950 and the compiler does not arrange by itself.
struct Unpack {
    uint32_t mask, one;
    __device__ Unpack()
    {
        asm volatile("v_mov_b32 %0, 0x03c003c0" : "=v"(mask));
        asm volatile("v_mov_b32 %0, 0x3c003c00" : "=v"(one));
    }
    __device__ v8h operator()(uint32_t w) const
    {
        v4i u;
        u[0] = (int)(((w << 6) & mask) | one);
        u[1] = (int)(((w << 2) & mask) | one);
        u[2] = (int)(((w >> 2) & mask) | one);
        u[3] = (int)(((w >> 6) & mask) | one);
        return __builtin_bit_cast(v8h, u);
    }
};

// fp16(p * s), s the low half of w: one v_fma_mixlo_f16 or v_fma_mixhi_f16, which round the
// product once.  Not in inline asm: the results are operands of matrix instructions, which
// may read them two wait states later at the earliest, and the compiler keeps that distance
// only from instructions that it sees.
__device__ __forceinline__ _Float16 scaled(float p, uint32_t w)
{
    return (_Float16)(p * (float)__builtin_bit_cast(_Float16, (uint16_t)w));
}

__device__ __forceinline__ v4f mfma16(v8h a, v8h b, v4f c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Reductions over the four lanes of one column (lane % 16): by swaps of the wave's
// halves and of its quarters.
template <class Op>
__device__ __forceinline__ float column_reduce(float v, Op op)
{
    uint32_t u = __float_as_uint(v);
    auto     r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    v          = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
    u          = __float_as_uint(v);
    r          = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return op(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ float column_max(float v)
{
    return column_reduce(v, [](float a, float b) { return fmaxf(a, b); });
}

__device__ __forceinline__ float column_sum(float v)
{
    return column_reduce(v, [](float a, float b) { return a + b; });
}

__device__ __forceinline__ float low_half(uint32_t w) { return half_bits_to_float(w & 0xFFFFu); }
__device__ __forceinline__ float high_half(uint32_t w) { return half_bits_to_float(w >> 16); }

// How the launch is cut: `waves` runs over all chunks, or (whole) over all units.
// Partials: slot 2 w + 0 of wave w holds a unit that began before its run, 2 w + 1 one
// that begins in it and goes on behind it: per head the sum of p v (fp32 [D]), then
// all slots' (maximum in powers of two, sum of p); then per unit the first wave of a
// cut one plus 1 (0: not cut) and the last.
struct Cut {
    uint32_t  waves, heads; // heads: query heads of a unit
    bool      whole;
    float*    o;
    float*    ml;
    uint32_t* unit;
};

__host__ __device__ inline uint32_t chunks_of(uint32_t len)
{
    return len == 0 ? 1u : (len + kChunk - 1) / kChunk; // a sequence of no tokens is written too
}

template <int D, int G>
struct KvLds {
    static constexpr int kGroups = D / G;
    static constexpr int kCodes  = kChunk * D / 2;       // bytes of a chunk's value codes
    static constexpr int kScales = kChunk * kGroups * 4; // bytes of its (scale, offset) pairs
    static constexpr int kWave   = kCodes + 2 * kScales; // value codes, key scales, value scales
};

// A chunk on its way: key codes as the product takes them, value codes as they go to
// LDS, and lane = token the (scale, offset) pairs.
template <int NG>
struct Chunk {
    v4i      k[4], v[4];
    int32_t  ks[NG], vs[NG];
    uint32_t ok; // which of its 16-token tiles have a page
};

// A chunk's place: sequence, unit of it, chunk of the unit (all wave-uniform).
struct Place {
    uint32_t seq, unit, chunk, chunks, len;
};

// N dwords, N = 1, 2 or 4, from global memory or to LDS in one access.
template <int N>
__device__ __forceinline__ void load_dwords(int32_t* r, const void* p)
{
    if constexpr(N == 4) {
        const v4i u = *static_cast<const v4i*>(p);
#pragma unroll
        for(int i = 0; i < 4; ++i) r[i] = u[i];
    } else if constexpr(N == 2) {
        const v2i u = *static_cast<const v2i*>(p);
        r[0] = u[0];
        r[1] = u[1];
    } else
        r[0] = *static_cast<const int32_t*>(p);
}

template <int N>
__device__ __forceinline__ void store_lds(uint32_t to, const int32_t* r)
{
    if constexpr(N == 4)
        *(lds_v4i_t*)(uintptr_t)to = v4i{r[0], r[1], r[2], r[3]};
    else if constexpr(N == 2)
        *(lds_v2i_t*)(uintptr_t)to = v2i{r[0], r[1]};
    else
        *(lds_u32_t*)(uintptr_t)to = (uint32_t)r[0];
}

template <int D, int G, int C>
__device__ __forceinline__ void attention_kv4_run(const CacheView& c, const AttentionKv4Args& a,
                                                  const Cut& cut, uint32_t pages, uint8_t* lds)
{
    using L              = KvLds<D, G>;
    constexpr int kSteps = D / 32, kPer = G / 32, kNG = D / G; // MFMA steps: all, per group
    constexpr int kTiles = D / 16;                             // channel tiles of the result
    constexpr int kHeads = kCols / C;                          // query heads of a unit
    constexpr int kPasses = 4 / C; // of the chunk's tiles: pass w takes tiles w C .. w C + C - 1
    constexpr int kRegs   = 4 * kPasses; // scores a lane holds: register 4 w + j is token
                                         // 16 (w C + class) + 4 kg + j
    const int      wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int      lane = threadIdx.x % kWave, col = lane % 16, kg = lane / 16;
    const int      cls = col / kHeads;
    const uint32_t run = blockIdx.x * kAttWaves + wave;
    if(run >= cut.waves) return;
    const uint32_t per = a.heads / c.kv_heads, qtiles = (per + kHeads - 1) / kHeads;
    const uint32_t units = c.kv_heads * qtiles; // of a sequence
    const uint32_t most  = a.table_cols * c.page_size;
    auto           length = [&](uint32_t seq) {
        return (uint32_t)max(0, (int)min((int64_t)a.lens[seq], (int64_t)most));
    };

    // ---- the wave's run ------------------------------------------------------------
    Place    here{0, 0, 0, 1, 0};
    uint32_t left = 0; // chunks of the run
    uint32_t q = 0, r = 0;
    if(cut.whole) {
        const uint32_t all = a.seqs * units;
        uint32_t       u   = (uint32_t)((uint64_t)run * all / cut.waves);
        const uint32_t to  = (uint32_t)((uint64_t)(run + 1) * all / cut.waves);
        here.seq           = u / units;
        here.unit          = u % units;
        for(; u < to; ++u) left += chunks_of(length(u / units));
    } else {
        auto scan = [&](uint32_t i0, uint32_t& n, uint32_t& s) { // 64 sequences' chunks
            const uint32_t i = i0 + lane;
            n                = i < a.seqs ? chunks_of(length(i)) * units : 0;
            s                = n;
#pragma unroll
            for(int d = 1; d < kWave; d <<= 1) {
                const uint32_t o = __shfl_up(s, d, kWave);
                if(lane >= d) s += o;
            }
            return (uint32_t)__builtin_amdgcn_readlane(s, kWave - 1);
        };
        uint32_t n, s, all = 0;
        for(uint32_t i = 0; i < a.seqs; i += kWave) all += scan(i, n, s);
        q                  = all / cut.waves;
        r                  = all % cut.waves;
        uint32_t       at  = run * q + min(run, r);
        left               = q + (run < r ? 1 : 0);
        if(left != 0)
            for(uint32_t i = 0; i < a.seqs; i += kWave) {
                const uint32_t sum = scan(i, n, s);
                if(at < sum) {
                    const int f = __builtin_ctzll(__ballot(s > at));
                    at -= __builtin_amdgcn_readlane(s, f) - __builtin_amdgcn_readlane(n, f);
                    here.seq = i + f;
                    break;
                }
                at -= sum;
            }
        here.chunk = at;
    }
    here.len    = left != 0 ? length(here.seq) : 0;
    here.chunks = chunks_of(here.len);
    if(!cut.whole) {
        here.unit  = here.chunk / here.chunks;
        here.chunk = here.chunk % here.chunks;
    }
    if(left == 0) return;
    auto advance = [&](Place& p) { // to the next chunk, whichever unit's; not past the run
        if(++p.chunk != p.chunks) return;
        p.chunk = 0;
        if(++p.unit != units) return;
        p.unit   = 0;
        p.seq    = min(p.seq + 1, a.seqs - 1);
        p.len    = length(p.seq);
        p.chunks = chunks_of(p.len);
    };

    // ---- chunks on their way ---------------------------------------------------------
    // a lane's bytes of a 16-token tile: of the keys 16 (8) of token lane % 16, of the
    // values 16 (8) of token lane / 4, which go to LDS with the 16-byte chunks of a row
    // swapped so that the transposed reads spread over the banks
    constexpr int  kBytes = D / 8;
    const uint32_t at     = (uint32_t)(uintptr_t)lds + wave * L::kWave;
    const uint32_t koff = lane % 16 * (D / 2) + kg * kBytes, voff = lane * kBytes;
    auto           row_chunk = [](uint32_t tok, uint32_t x) {
        return x ^ (D == 128 ? tok / 4 % 4 : tok / 8 % 2);
    };
    const uint32_t vto = at + lane / 4 * (D / 2)
                         + row_chunk(lane / 4, lane % 4 * kBytes / 16) * 16 + lane % 4 * kBytes % 16;
    auto page_at = [&](const Place& p) { // lane / 16 = tile: its page, or -1
        const uint32_t t    = p.chunk * kChunk + lane / 16 * 16;
        int32_t        page = -1;
        if(t < p.len) {
            page = a.table[(size_t)p.seq * a.table_ld + (t >> c.page_shift)];
            if(page < 0 || (uint32_t)page >= pages) page = -1;
        }
        return page;
    };
    // byte offset of the codes of tile i of a chunk; a tile without a page reads page 0's
    // rows and is masked
    auto tile_codes = [&](const Place& p, int32_t page, int i) {
        const int32_t g = __builtin_amdgcn_readlane(page, 16 * i);
        return cache_row(c, g >= 0 ? g : 0, p.unit / qtiles,
                         (p.chunk * kChunk + i * 16) & (c.page_size - 1))
               * (D / 2);
    };
    auto fetch_values = [&](Chunk<kNG>& x, const Place& p, int32_t page) {
        const uint64_t with = __ballot(page >= 0);
        x.ok = (uint32_t)(with & 1) | (uint32_t)(with >> 15 & 2) | (uint32_t)(with >> 30 & 4)
               | (uint32_t)(with >> 45 & 8);
        const size_t mine = cache_row(c, page >= 0 ? page : 0, p.unit / qtiles, // lane = token
                                      (p.chunk * kChunk + lane) & (c.page_size - 1));
#pragma unroll
        for(int i = 0; i < 4; ++i)
            load_dwords<D / 32>(reinterpret_cast<int32_t*>(&x.v[i]),
                                c.codes[1] + tile_codes(p, page, i) + voff);
        load_dwords<kNG>(x.ks, c.scales[0] + mine * kNG);
        load_dwords<kNG>(x.vs, c.scales[1] + mine * kNG);
    };
    auto fetch_keys = [&](Chunk<kNG>& x, const Place& p, int32_t page) {
#pragma unroll
        for(int i = 0; i < 4; ++i)
            load_dwords<D / 32>(reinterpret_cast<int32_t*>(&x.k[i]),
                                c.codes[0] + tile_codes(p, page, i) + koff);
    };

    // ---- the queries: column = head, 8 channels a step in the codes' order -----------
    v8h   qf[C][kSteps]; // zero but for the lane's own class
    float mid[kNG];      // 1.5 times the sum of the group's channels
    float qsum[kNG];     // the sum / 16
    auto  queries = [&](const Place& p) {
        const uint32_t  first = p.unit % qtiles * kHeads, h = first + col % kHeads;
        const uint16_t* from  = a.q + (size_t)p.seq * a.ldq
                               + (size_t)(p.unit / qtiles * per + min(h, per - 1)) * D + 8 * kg;
        constexpr int kOrder[8] = {0, 4, 1, 5, 2, 6, 3, 7};
        v8h           v[kSteps];
#pragma unroll
        for(int j = 0; j < kSteps; ++j) v[j] = *reinterpret_cast<const v8h*>(from + 32 * j);
#pragma unroll
        for(int g = 0; g < kNG; ++g) {
            float sum = 0.f;
#pragma unroll
            for(int j = g * kPer; j < (g + 1) * kPer; ++j) {
                v8h u;
#pragma unroll
                for(int e = 0; e < 8; ++e) {
                    u[e] = v[j][kOrder[e]];
                    sum += (float)v[j][e];
                }
#pragma unroll
                for(int x = 0; x < C; ++x) qf[x][j] = cls == x ? u : v8h{};
            }
            sum      = column_sum(sum);
            qsum[g]  = sum * 0.0625f;
            mid[g]   = sum * 1.5f;
        }
    };

    const Unpack unpack;
    const float  c2 = a.scale * (16.f * 1.44269504088896341f); // scores are held / 16
    // of the operand of O^T: which halves hold the lane's class in products 0 and 1
    const uint32_t half = cls % 2 == 0 ? 0xFFFFu : 0xFFFF0000u;
    const uint32_t half_mask[2]
        = {C < 4 || cls / 2 == 0 ? half : 0u, C < 4 || cls / 2 == 1 ? half : 0u};

    float m = -INFINITY, l = 0.f;
    int   shift = 0; // p s is held times 2^shift
    v4f   o[kTiles] = {}, total[kNG] = {};
    float osum[kNG] = {};
    bool  from_start = here.chunk == 0; // of the unit

    Chunk<kNG> x;
    Place      next = here;
    {
        const int32_t page = page_at(here);
        queries(here);
        fetch_values(x, here, page);
        fetch_keys(x, here, page);
    }
    int32_t page_next = -1;
    if(left > 1) {
        advance(next);
        page_next = page_at(next);
    }

    for(; left > 0; --left) {
        const uint32_t t0   = here.chunk * kChunk;
        const uint32_t live = x.ok;
        const bool     full = live == 15u && t0 + kChunk <= here.len;
        if(!full && (t0 + lane >= here.len || !((live >> (lane / 16)) & 1u)))
#pragma unroll
            for(int g = 0; g < kNG; ++g) x.vs[g] = 0; // not there: it may be NaN
#pragma unroll
        for(int i = 0; i < 4; ++i)
            store_lds<D / 32>(vto + i * 16 * (D / 2), reinterpret_cast<const int32_t*>(&x.v[i]));
        store_lds<kNG>(at + L::kCodes + lane * kNG * 4, x.ks);
        store_lds<kNG>(at + L::kCodes + L::kScales + lane * kNG * 4, x.vs);
        float big = 0.f; // the largest scale of the values
#pragma unroll
        for(int g = 0; g < kNG; ++g) big = fmaxf(big, fabsf(low_half((uint32_t)x.vs[g])));
        big = wave_max(big);
        v4i k[4]; // this chunk's: x is the next one's from here on
#pragma unroll
        for(int i = 0; i < 4; ++i) k[i] = x.k[i];
        const Place now = here;
        if(left > 1) {
            const int32_t page = page_next;
            here               = next;
            if(left > 2) {
                advance(next);
                page_next = page_at(next);
            }
            fetch_values(x, here, page);
            fetch_keys(x, here, page);
        }

        // ---- scores -----------------------------------------------------------------
        float s[kRegs];
#pragma unroll
        for(int w = 0; w < kPasses; ++w) {
            v4i sk[kNG];
#pragma unroll
            for(int g = 0; g < kNG; ++g)
                sk[g] = *(const lds_v4i_t*)(uintptr_t)(
                    at + L::kCodes + (16 * (w * C + cls) + 4 * kg) * kNG * 4 + g * 16);
#pragma unroll
            for(int g = 0; g < kNG; ++g) {
                v4f acc = {};
#pragma unroll
                for(int y = 0; y < C; ++y)
#pragma unroll
                    for(int j = g * kPer; j < (g + 1) * kPer; ++j)
                        acc = mfma16(unpack((uint32_t)k[w * C + y][j]), qf[y][j], acc);
#pragma unroll
                for(int j = 0; j < 4; ++j) {
                    const uint32_t u = (uint32_t)sk[(j * kNG + g) / 4][(j * kNG + g) % 4];
                    const float    b = g == 0 ? 0.f : s[4 * w + j];
                    s[4 * w + j]
                        = fmaf(low_half(u), acc[j] - mid[g], fmaf(high_half(u), qsum[g], b));
                }
            }
        }
        if(!full) // tokens that are not there
#pragma unroll
            for(int i = 0; i < kRegs; ++i) {
                const uint32_t tile = i / 4 * C + cls;
                if(t0 + 16 * tile + 4 * kg + i % 4 >= now.len || !((live >> tile) & 1u))
                    s[i] = -INFINITY;
            }
        // ---- the power of two that goes with the largest scale ------------------------
        float       rescale = 1.f;
        const float held    = ldexpf(big, shift);
        if(big > 0.f && big <= 65504.f && (held < 1.f || held > 64.f)) {
            const int to = 4 - __builtin_amdgcn_frexp_expf(big);
            rescale      = ldexpf(1.f, to - shift);
            shift        = to;
        }

        // ---- softmax ------------------------------------------------------------------
        float top = s[0];
#pragma unroll
        for(int i = 1; i < kRegs; ++i) top = fmaxf(top, s[i]);
        const float mn = fmaxf(m, column_max(top));
        if(__ballot(mn > m) != 0 || rescale != 1.f) {
            const float al = m == mn ? 1.f : __builtin_amdgcn_exp2f((m - mn) * c2);
            m              = mn;
            l *= al;
#pragma unroll
            for(int g = 0; g < kNG; ++g) {
                osum[g] *= al;
                total[g] *= al * rescale;
            }
#pragma unroll
            for(int t = 0; t < kTiles; ++t) o[t] *= al * rescale;
        }
        const float mc = m == -INFINITY ? 0.f : m * c2; // no token yet: every p is 0
        float       p[kRegs];
#pragma unroll
        for(int i = 0; i < kRegs; ++i) {
            p[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c2, -mc));
            l += p[i];
        }

        // ---- p times the values' scales, as the operand, group by group ----------------
        // operand register r of product u: token 4 kg + r of tile 2 u in the low and of
        // tile 2 u + 1 in the high half, zero for tiles of other classes
        const float pow2 = ldexpf(1.f, shift);
        v2h         ps[kNG][2][4];
#pragma unroll
        for(int w = 0; w < kPasses; ++w) {
            v4i sv[kNG];
#pragma unroll
            for(int g = 0; g < kNG; ++g)
                sv[g] = *(const lds_v4i_t*)(uintptr_t)(
                    at + L::kCodes + L::kScales + (16 * (w * C + cls) + 4 * kg) * kNG * 4 + g * 16);
#pragma unroll
            for(int j = 0; j < 4; ++j) {
                const float f = p[4 * w + j] * pow2;
#pragma unroll
                for(int g = 0; g < kNG; ++g) {
                    const uint32_t u = (uint32_t)sv[(j * kNG + g) / 4][(j * kNG + g) % 4];
                    osum[g]          = fmaf(p[4 * w + j], high_half(u), osum[g]);
                    const _Float16 h = scaled(f, u);
                    if constexpr(C == 1)
                        ps[g][w / 2][j][w % 2] = h;
                    else {
                        const uint32_t b = __builtin_bit_cast(uint32_t, (v2h{h, h}));
                        if constexpr(C == 2)
                            ps[g][w][j] = __builtin_bit_cast(v2h, b & half_mask[0]);
                        else
#pragma unroll
                            for(int y = 0; y < 2; ++y)
                                ps[g][y][j] = __builtin_bit_cast(v2h, b & half_mask[y]);
                    }
                }
            }
        }
        auto operand = [&](int g, int u) {
            v8h f;
#pragma unroll
            for(int i = 0; i < 8; ++i) f[i] = ps[g][u][i / 2][i % 2];
            return f;
        };
        const v8h ones = {1, 1, 1, 1, 1, 1, 1, 1};
#pragma unroll
        for(int g = 0; g < kNG; ++g)
#pragma unroll
            for(int u = 0; u < 2; ++u) total[g] = mfma16(ones, operand(g, u), total[g]);

        // ---- values: channel 16 t + col, tokens of source lanes 16 (j / 4) + 4 kg + j % 4
#pragma unroll
        for(int t = 0; t < kTiles; ++t) {
            const uint32_t tok = 16 * (col / 4) + 4 * kg + col % 4;
            const v2i      w   = __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_v2i_t*)(uintptr_t)(
                at + tok * (D / 2) + row_chunk(tok, t / 2) * 16 + t % 2 * 8));
#pragma unroll
            for(int u = 0; u < 2; ++u)
                o[t] = mfma16(unpack((uint32_t)w[u]), operand(t * 16 / G, u), o[t]);
        }

        // ---- the unit's end, or the run's -----------------------------------------------
        const bool ends = now.chunk + 1 == now.chunks;
        if(!ends && left > 1) continue;
        // classes side by side: a common maximum, then sums over the columns of a head
        l            = column_sum(l);
        float common = m;
        if constexpr(C >= 4) common = fmaxf(common, dpp_mov<kDppRowRor4>(common));
        if constexpr(C >= 2) common = fmaxf(common, dpp_mov<kDppRowRor8>(common));
        const float f = l == 0.f ? 0.f : m == common ? 1.f : __builtin_amdgcn_exp2f((m - common) * c2);
        auto        merged = [&](float v) {
            v *= f;
            if constexpr(C >= 4) v += dpp_mov<kDppRowRor4>(v);
            if constexpr(C >= 2) v += dpp_mov<kDppRowRor8>(v);
            return v;
        };
        l                  = merged(l);
        const float    back = ldexpf(16.f, -shift);
        const uint32_t head = now.unit % qtiles * kHeads + col; // of the key head's
        const bool     mine = cls == 0 && head < per;
        const bool     done = ends && from_start;
        const float    inv  = done ? (l != 0.f ? 1.f / l : 0.f) : 1.f;
        const uint32_t slot = 2 * run + (from_start ? 1 : 0);
#pragma unroll
        for(int g = 0; g < kNG; ++g) osum[g] = column_sum(osum[g]);
#pragma unroll
        for(int t = 0; t < kTiles; ++t) {
            const int g = t * 16 / G;
            v4f       v;
#pragma unroll
            for(int i = 0; i < 4; ++i)
                v[i] = merged(fmaf(fmaf(total[g][i], -1.5f, o[t][i]), back, osum[g])) * inv;
            if(!mine) continue;
            if(done) {
                const size_t to = (size_t)now.seq * a.ldo
                                  + (size_t)(now.unit / qtiles * per + head) * D + 16 * t + 4 * kg;
                v2i w;
                w[0] = (int)finite_halves(v[0], v[1]);
                w[1] = (int)finite_halves(v[2], v[3]);
                *reinterpret_cast<v2i*>(a.out + to) = w;
            } else
                *reinterpret_cast<v4f*>(cut.o + ((size_t)slot * kHeads + col) * D + 16 * t + 4 * kg)
                    = v;
        }
        if(!done && mine && kg == 0) {
            cut.ml[((size_t)slot * kHeads + col) * 2]     = common * c2;
            cut.ml[((size_t)slot * kHeads + col) * 2 + 1] = l;
        }
        if(from_start && !cut.whole && lane == 0) {
            uint32_t* to = cut.unit + 2 * ((size_t)now.seq * units + now.unit);
            to[0]        = ends ? 0 : run + 1;
            if(!ends) { // goes on behind the run: up to which wave
                const uint32_t end  = run * q + min(run, r) + (q + (run < r ? 1 : 0));
                const uint32_t last = end + (now.chunks - 1 - now.chunk) - 1; // its last chunk
                to[1] = last < r * (q + 1) ? last / (q + 1) : r + (last - r * (q + 1)) / q;
            }
        }
        if(left > 1) { // the next unit
            from_start = true;
            m          = -INFINITY;
            l          = 0.f;
#pragma unroll
            for(int g = 0; g < kNG; ++g) {
                osum[g]  = 0.f;
                total[g] = v4f{0, 0, 0, 0};
            }
#pragma unroll
            for(int t = 0; t < kTiles; ++t) o[t] = v4f{0, 0, 0, 0};
            queries(here);
        }
    }
}

template <int D, int G, int C>
__global__ void __launch_bounds__(kAttThreads, 2)
    attention_kv4_kernel(CacheView c, AttentionKv4Args a, Cut cut, uint32_t pages)
{
    __shared__ alignas(16) uint8_t lds[kAttWaves * KvLds<D, G>::kWave];
    attention_kv4_run<D, G, C>(c, a, cut, pages, lds);
}

// Joins the partials of the cut units: the slot of the first wave, then the first slots
// of the waves after it.  WAVES waves take CH channels of one head of a unit, CH / 4
// lanes 4 channels each of every kWays-th partial, 8 loads at a time with a running
// maximum; then the ways are added up, always in the same order.  Few units have many
// partials each and take all of a block's waves for a part of the channels (1 x 131072
// tokens, 8 key heads: 256 partials a unit), many units have few and take a wave a head.
// Blocks are kept few: their start is what a launch of thousands waits for.
template <int D, int HEADS, int WAVES, int CH>
__global__ void __launch_bounds__(kAttThreads)
    attention_kv4_join_kernel(AttentionKv4Args a, Cut cut, uint32_t kv_heads, uint32_t tasks)
{
    constexpr uint32_t kLanes = CH / 4, kWays = WAVES * kWave / kLanes, kSlices = D / CH;
    constexpr uint32_t kGroups = kAttWaves / WAVES;
    __shared__ v4f   part[WAVES][kLanes];
    __shared__ float top[WAVES], weight[WAVES];
    const int        wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t   lane = threadIdx.x % kWave, in = threadIdx.x % (WAVES * kWave);
    const uint32_t   way = in / kLanes;
    const uint32_t   per = a.heads / kv_heads, qtiles = (per + HEADS - 1) / HEADS;
    const uint32_t   units = kv_heads * qtiles; // of a sequence
    for(uint32_t task = blockIdx.x * kGroups + wave / WAVES; task < tasks;
        task += gridDim.x * kGroups) {
        const uint32_t u = task / (HEADS * kSlices), col = task / kSlices % HEADS;
        const uint32_t ch = task % kSlices * CH + in % kLanes * 4;
        const uint32_t w0 = __builtin_amdgcn_readfirstlane(cut.unit[2 * (size_t)u]);
        const uint32_t w1 = __builtin_amdgcn_readfirstlane(cut.unit[2 * (size_t)u + 1]);
        const uint32_t head = u % units % qtiles * HEADS + col;
        if(w0 == 0 || head >= per) continue;
        const uint32_t run = w0 - 1, n = w1 - run + 1; // partials
        float          m = -INFINITY, l = 0.f;
        v4f            sum = {};
        auto take = [&](float mi, float li, v4f v) { // 0: no token seen, its maximum is -inf
            if(li == 0.f) return;
            const float now = fmaxf(m, mi);
            const float al  = m == now ? 1.f : __builtin_amdgcn_exp2f(m - now);
            const float e   = mi == now ? 1.f : __builtin_amdgcn_exp2f(mi - now);
            m               = now;
            l               = fmaf(l, al, e * li);
#pragma unroll
            for(int y = 0; y < 4; ++y) sum[y] = fmaf(sum[y], al, e * v[y]);
        };
        for(uint32_t i0 = way; i0 < n; i0 += 8 * kWays) {
            v4f v[8];
            v2f ml[8];
#pragma unroll
            for(int x = 0; x < 8; ++x) {
                const uint32_t i    = min(i0 + x * kWays, n - 1);
                const size_t   from = (size_t)(2 * (run + i) + (i == 0 ? 1 : 0)) * HEADS + col;
                v[x]  = *reinterpret_cast<const v4f*>(cut.o + from * D + ch);
                ml[x] = *reinterpret_cast<const v2f*>(cut.ml + from * 2);
            }
#pragma unroll
            for(int x = 0; x < 8; ++x) take(ml[x][0], i0 + x * kWays < n ? ml[x][1] : 0.f, v[x]);
        }
#pragma unroll
        for(int d = kLanes; d < kWave; d <<= 1) { // the ways of a wave, in pairs
            const float mo = __shfl_xor(m, d, kWave), lo = __shfl_xor(l, d, kWave);
            v4f         vo;
#pragma unroll
            for(int y = 0; y < 4; ++y) vo[y] = __shfl_xor(sum[y], d, kWave);
            take(mo, lo, vo);
        }
        if constexpr(WAVES > 1) { // one task a block: its waves come here together
            __syncthreads();
            if(lane < kLanes) part[wave][lane] = sum;
            if(lane == 0) {
                top[wave]    = m;
                weight[wave] = l;
            }
            __syncthreads();
            m   = -INFINITY;
            l   = 0.f;
            sum = v4f{0, 0, 0, 0};
#pragma unroll
            for(int w = 0; w < WAVES; ++w) take(top[w], weight[w], part[w][in % kLanes]);
        }
        if(way != 0) continue;
        const float inv = l != 0.f ? 1.f / l : 0.f;
        v2i         w;
        w[0] = (int)finite_halves(sum[0] * inv, sum[1] * inv);
        w[1] = (int)finite_halves(sum[2] * inv, sum[3] * inv);
        *reinterpret_cast<v2i*>(a.out + (size_t)(u / units) * a.ldo
                                + (size_t)(u % units / qtiles * per + head) * D + ch)
            = w;
    }
}

template <int D, int HEADS>
void launch_join(const AttentionKv4Args& a, const Cut& cut, uint32_t kv_heads, uint32_t units,
                 hipStream_t stream)
{
    constexpr uint32_t kMostBlocks = 1024;
    const uint32_t     heads = a.seqs * units * HEADS;
    if(heads <= 256)
        attention_kv4_join_kernel<D, HEADS, kAttWaves, 32>
            <<<heads * (D / 32), kAttThreads, 0, stream>>>(a, cut, kv_heads, heads * (D / 32));
    else
        attention_kv4_join_kernel<D, HEADS, 1, D>
            <<<std::min((heads + kAttWaves - 1) / kAttWaves, kMostBlocks), kAttThreads, 0, stream>>>(
                a, cut, kv_heads, heads);
}

// Query heads a unit takes: all of a key head's where they are few.
uint32_t unit_heads(uint32_t per) { return per <= 4 ? 4 : per <= 8 ? 8 : 16; }

uint32_t seq_units(uint32_t heads, uint32_t kv_heads)
{
    const uint32_t per = heads / kv_heads, b = unit_heads(per);
    return kv_heads * ((per + b - 1) / b);
}

// Waves of the launch: no more than chunks at the most.
uint32_t run_count(uint32_t seqs, uint32_t units, uint32_t max_len)
{
    return (uint32_t)std::min<uint64_t>(kAttBlocks * kAttWaves,
                                        (uint64_t)seqs * units * chunks_of(max_len));
}

} // namespace

hipError_t launch_kv4_store(const w8a8_kv4_cache& c, const Kv4Rows& r, const uint16_t* k,
                            const uint16_t* v, hipStream_t stream)
{
    with_widths(c, [&](auto d, auto g) {
        const RowPlan p = row_plan(c, r);
        kv4_store_kernel<d(), g()><<<p.blocks, kRowThreads, 0, stream>>>(view(c), r, p, k, v);
    });
    return hipGetLastError();
}

hipError_t launch_kv4_load(const w8a8_kv4_cache& c, const Kv4Rows& r, uint16_t* k, uint16_t* v,
                           hipStream_t stream)
{
    with_widths(c, [&](auto d, auto g) {
        const RowPlan p = row_plan(c, r);
        kv4_load_kernel<d(), g()><<<p.blocks, kRowThreads, 0, stream>>>(view(c), r, p, k, v);
    });
    return hipGetLastError();
}

size_t attention_kv4_workspace_bytes(uint32_t seqs, uint32_t heads, uint32_t kv_heads, uint32_t dim,
                                     uint32_t max_len)
{
    if(chunks_of(max_len) == 1) return 0; // no unit is cut
    const size_t waves = run_count(seqs, seq_units(heads, kv_heads), max_len);
    return waves * 2 * unit_heads(heads / kv_heads) * (dim + 2) * 4
           + (size_t)seqs * seq_units(heads, kv_heads) * 8;
}

hipError_t launch_attention_kv4(const w8a8_kv4_cache& c, const AttentionKv4Args& a,
                                hipStream_t stream)
{
    const uint32_t max_len = a.table_cols * c.page_size, units = seq_units(a.heads, c.kv_heads);
    const size_t   need
        = attention_kv4_workspace_bytes(a.seqs, a.heads, c.kv_heads, c.head_dim, max_len);
    Cut cut{};
    cut.heads = unit_heads(a.heads / c.kv_heads);
    cut.whole = need == 0 || a.ws_bytes < need;
    if(cut.whole)
        cut.waves = std::min(kAttBlocks * kAttWaves, a.seqs * units);
    else {
        cut.waves          = run_count(a.seqs, units, max_len);
        const size_t slots = (size_t)cut.waves * 2 * cut.heads;
        cut.o              = static_cast<float*>(a.ws);
        cut.ml             = cut.o + slots * c.head_dim;
        cut.unit           = reinterpret_cast<uint32_t*>(cut.ml + slots * 2);
    }
    const uint32_t blocks = (cut.waves + kAttWaves - 1) / kAttWaves;
    with_widths(c, [&](auto d, auto g) {
        const auto kernel = cut.heads == 4   ? attention_kv4_kernel<d(), g(), 4>
                            : cut.heads == 8 ? attention_kv4_kernel<d(), g(), 2>
                                             : attention_kv4_kernel<d(), g(), 1>;
        kernel<<<blocks, kAttThreads, 0, stream>>>(view(c), a, cut, c.pages);
        if(!cut.whole) {
            const auto join = cut.heads == 4   ? launch_join<d(), 4>
                              : cut.heads == 8 ? launch_join<d(), 8>
                                               : launch_join<d(), 16>;
            join(a, cut, c.kv_heads, units, stream);
        }
    });
    return hipGetLastError();
}

} // namespace w8a8
