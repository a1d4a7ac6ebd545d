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

// ---------------------------------------------------------------------------
// Attention of single tokens over the cache.
//
// A block owns a piece of one sequence's context for the (up to 16) query heads of
// one key head; its waves take chunks of 64 tokens in turn, each with its own
// running maximum and sum, and merge at the end.  Both products run on
// v_mfma_f32_16x16x32_f16 with the query heads as columns:
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
// (the -1.5 makes x the centred code; in S^T it is the accumulator's start, in O^T
// the sum over the tokens of the rounded p s, from a matrix product with ones, so
// that rounding p s to fp16, the only rounding below fp32, acts on the centred
// code).  p s is brought to fp16's range by a power of two that follows the scales.
// ---------------------------------------------------------------------------
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float    v2f __attribute__((ext_vector_type(2)));

typedef __attribute__((address_space(3))) v2i      lds_v2i_t;
typedef __attribute__((address_space(3))) v4i      lds_v4i_t;
typedef __attribute__((address_space(3))) uint32_t lds_u32_t;

constexpr int kAttWaves   = 4;
constexpr int kAttThreads = kAttWaves * kWave;
constexpr int kChunk      = 64;   // tokens a wave takes at a time
constexpr int kSegment    = 4096; // tokens whose page numbers lie in LDS at a time
constexpr int kCols       = 16;   // query heads a block takes

// `size` 16 or 4 bytes a lane from base + offset into LDS, lane i to `to` + size * i,
// with the caller's own wait (the builtin makes the compiler wait for every such
// load ahead of each transposed read).
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm" // m0 is reserved: set and used here alone
template <int SIZE>
__device__ __forceinline__ void load_lds(const void* base, uint32_t to, uint32_t offset)
{
    if constexpr(SIZE == 16)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                     :
                     : "s"(to), "v"(offset), "s"(base)
                     : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
                     :
                     : "s"(to), "v"(offset), "s"(base)
                     : "memory", "m0");
}
#pragma clang diagnostic pop

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

// fp16(p0 * s0) and fp16(p1 * s1), s the low halves of w0 and w1, as a packed pair:
// each product rounded once, in one instruction.
__device__ __forceinline__ uint32_t scaled_pair(float p0, uint32_t w0, float p1, uint32_t w1)
{
    uint32_t r;
    asm("v_fma_mixlo_f16 %0, %1, %2, 0 op_sel_hi:[0,1,0]" : "=v"(r) : "v"(p0), "v"(w0));
    asm("v_fma_mixhi_f16 %0, %1, %2, 0 op_sel_hi:[0,1,0]" : "+v"(r) : "v"(p1), "v"(w1));
    return r;
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

// Pieces a sequence's context is cut into, and where they leave their results:
// per (sequence, head) and piece the sum of p v (fp32 [D]), the maximum in powers
// of two and the sum of p.
struct Pieces {
    uint32_t count, tokens;
    float*   o;
    float*   ml;
};

template <int D, int G>
struct KvLds {
    static constexpr int kGroups = D / G;
    static constexpr int kCodes  = kChunk * D / 2;        // bytes of a chunk's value codes
    static constexpr int kScales = kChunk * kGroups * 4;  // bytes of its (scale, offset) pairs
    static constexpr int kStage  = kCodes + 2 * kScales;  // value codes, key scales, value scales
    static constexpr int kRing   = kAttWaves * 2 * kStage;
    static constexpr int kMerge  = kAttWaves * kCols * (D + 2) * 4;
    static constexpr int kBytes  = kRing > kMerge ? kRing : kMerge;
};

template <int D, int G>
__device__ __forceinline__ void attention_kv4_piece(const CacheView& c, const AttentionKv4Args& a,
                                                    const Pieces& pieces, uint32_t pages,
                                                    uint8_t* lds, int32_t* page_of)
{
    using L              = KvLds<D, G>;
    constexpr int kSteps = D / 32, kPer = G / 32, kNG = D / G; // MFMA steps: all, per group
    constexpr int kTiles = D / 16;                             // channel tiles of the result
    const int      wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int      lane = threadIdx.x % kWave, col = lane % 16, kg = lane / 16;
    const uint32_t per = a.heads / c.kv_heads, qtiles = (per + kCols - 1) / kCols;
    const uint32_t kvh = blockIdx.x / qtiles, first = blockIdx.x % qtiles * kCols;
    const uint32_t seq = blockIdx.y, heads = min((uint32_t)kCols, per - first);
    const uint32_t head0 = kvh * per + first; // the block's first query head
    const uint32_t most  = a.table_cols * c.page_size;
    const uint32_t len   = (uint32_t)max(0, (int)min((int64_t)a.lens[seq], (int64_t)most));
    const uint32_t begin = blockIdx.z * pieces.tokens;
    const uint32_t end   = min(len, pieces.count == 1 ? most : begin + pieces.tokens);
    if(begin >= end && pieces.count > 1) return;

    // ---- the queries: column = head, 8 channels a step in the codes' order -------
    v8h   qf[kSteps];
    v4f   start[kNG]; // -1.5 times the sum of the group's channels
    float qsum[kNG];  // the sum / 16
    {
        const uint16_t* q = a.q + (size_t)seq * a.ldq + (size_t)(head0 + col) * D;
        constexpr int   kOrder[8] = {0, 4, 1, 5, 2, 6, 3, 7};
#pragma unroll
        for(int g = 0; g < kNG; ++g) {
            float sum = 0.f;
#pragma unroll
            for(int j = g * kPer; j < (g + 1) * kPer; ++j) {
                v8h v = {};
                if((uint32_t)col < heads)
                    v = *reinterpret_cast<const v8h*>(q + 32 * j + 8 * kg);
#pragma unroll
                for(int e = 0; e < 8; ++e) {
                    qf[j][e] = v[kOrder[e]];
                    sum += (float)v[e];
                }
            }
            sum      = column_sum(sum);
            qsum[g]  = sum * 0.0625f;
            start[g] = v4f{sum, sum, sum, sum} * -1.5f;
        }
    }

    const float    c2    = a.scale * (16.f * 1.44269504088896341f); // scores are held / 16
    const uint32_t lds0  = (uint32_t)(uintptr_t)lds;
    const uint32_t ring  = lds0 + wave * 2 * L::kStage;
    const size_t   row_k = (size_t)(lane % 16) * (D / 2) + kg * (D / 8);
    constexpr int  kRowChunks = D / 32; // 16-byte chunks of a row of codes
    const uint32_t vr = lane / kRowChunks, vp = lane % kRowChunks;
    const uint32_t voff = vr * (D / 2) + (vp ^ (D == 128 ? vr / 4 % 4 : vr / 8 % 2)) * 16;

    const Unpack unpack;
    float        m = -INFINITY, l = 0.f;
    int          shift = 0; // p s is held times 2^shift
    v4f   o[kTiles] = {}, total[kNG] = {};
    float osum[kNG] = {};

    for(uint32_t seg = begin; seg < end; seg += kSegment) {
        const uint32_t seg_end = min(end, seg + kSegment);
        __syncthreads();
        {
            const uint32_t t = seg + threadIdx.x * 16; // one page number per 16 tokens
            int32_t        p = -1;
            if(t < seg_end) {
                p = a.table[(size_t)seq * a.table_ld + (t >> c.page_shift)];
                if(p < 0 || (uint32_t)p >= pages) p = -1;
            }
            page_of[threadIdx.x] = p;
        }
        __syncthreads();

        v4i      kc[4];  // the key codes of the chunk ahead
        uint32_t ok = 0; // which of its 16-token tiles have a page
        auto     issue = [&](uint32_t chunk, uint32_t stage) {
            ok = 0;
#pragma unroll
            for(int i = 0; i < 4; ++i) {
                const uint32_t t = seg + chunk * kChunk + i * 16;
                const int32_t  p = __builtin_amdgcn_readfirstlane(page_of[chunk * 4 + i]);
                ok |= (p >= 0 ? 1u : 0u) << i;
                // a tile without a page reads page 0's rows and is masked
                const size_t row = cache_row(c, p >= 0 ? p : 0, kvh, t & (c.page_size - 1));
                const uint8_t* k = c.codes[0] + row * (D / 2) + row_k;
                if constexpr(D == 128)
                    kc[i] = *reinterpret_cast<const v4i*>(k);
                else {
                    const v2i u = *reinterpret_cast<const v2i*>(k);
                    kc[i]       = v4i{u[0], u[1], 0, 0};
                }
                const uint32_t to = ring + stage * L::kStage;
                if(lane < 16 * kRowChunks)
                    load_lds<16>(c.codes[1] + row * (D / 2), to + i * 16 * (D / 2), voff);
                if(lane < 16 * kNG) {
                    load_lds<4>(c.scales[0] + row * kNG, to + L::kCodes + i * 64 * kNG, lane * 4);
                    load_lds<4>(c.scales[1] + row * kNG, to + L::kCodes + L::kScales + i * 64 * kNG,
                                lane * 4);
                }
            }
        };

        const uint32_t chunks = (seg_end - seg + kChunk - 1) / kChunk;
        if((uint32_t)wave < chunks) issue(wave, 0);
        uint32_t stage = 0;
        for(uint32_t chunk = wave; chunk < chunks; chunk += kAttWaves, stage ^= 1) {
            wait_vmcnt<0>();  // the chunk is there,
            wait_lgkmcnt0();  // and the reads of the one before, whose stage is next, are done
            asm volatile("" ::: "memory");
            v4i kn[4];
#pragma unroll
            for(int i = 0; i < 4; ++i) kn[i] = kc[i];
            const uint32_t t0   = seg + chunk * kChunk;
            const uint32_t live = ok;
            const bool     full = live == 15u && t0 + kChunk <= end;
            if(chunk + kAttWaves < chunks) issue(chunk + kAttWaves, stage ^ 1);
            const uint32_t at = ring + stage * L::kStage;

            // ---- scores: register 4 i + j of a lane is token 16 i + 4 kg + j --------
            float s[16];
#pragma unroll
            for(int i = 0; i < 4; ++i) {
                v4i sk[kNG];
#pragma unroll
                for(int g = 0; g < kNG; ++g)
                    sk[g] = *(const lds_v4i_t*)(uintptr_t)(at + L::kCodes
                                                           + (16 * i + 4 * kg) * kNG * 4 + g * 16);
#pragma unroll
                for(int g = 0; g < kNG; ++g) {
                    v4f acc = start[g];
#pragma unroll
                    for(int j = g * kPer; j < (g + 1) * kPer; ++j)
                        acc = mfma16(unpack((uint32_t)kn[i][j]), qf[j], acc);
#pragma unroll
                    for(int j = 0; j < 4; ++j) {
                        const uint32_t w = (uint32_t)sk[(j * kNG + g) / 4][(j * kNG + g) % 4];
                        const float    x = g == 0 ? 0.f : s[4 * i + j];
                        s[4 * i + j]     = fmaf(low_half(w), acc[j], fmaf(high_half(w), qsum[g], x));
                    }
                }
            }
            if(!full) { // tokens that are not there: no score, and no scales (what lies there
                        // may be NaN)
#pragma unroll
                for(int r = 0; r < 16; ++r)
                    if(t0 + 16 * (r / 4) + 4 * kg + r % 4 >= end || !((live >> (r / 4)) & 1u))
                        s[r] = -INFINITY;
                if(t0 + lane >= end || !((live >> (lane / 16)) & 1u))
#pragma unroll
                    for(int g = 0; g < kNG; ++g)
                        *(lds_u32_t*)(uintptr_t)(at + L::kCodes + L::kScales + (lane * kNG + g) * 4)
                            = 0;
            }

            // ---- the largest scale of the values, and with it the power of two -----
            float big = 0.f;
#pragma unroll
            for(int g = 0; g < kNG; ++g)
                big = fmaxf(big, fabsf(low_half(*(const lds_u32_t*)(uintptr_t)(
                                     at + L::kCodes + L::kScales + (lane * kNG + g) * 4))));
            big = wave_max(big);
            float       rescale = 1.f;
            const float now     = ldexpf(big, shift);
            if(big > 0.f && big <= 65504.f && (now < 1.f || now > 64.f)) {
                const int next = 4 - __builtin_amdgcn_frexp_expf(big);
                rescale        = ldexpf(1.f, next - shift);
                shift          = next;
            }

            // ---- softmax -------------------------------------------------------
            float top = s[0];
#pragma unroll
            for(int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
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
            float       p[16];
#pragma unroll
            for(int r = 0; r < 16; ++r) {
                p[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c2, -mc));
                l += p[r];
            }

            // ---- p times the values' scales, as the operand, group by group --------
            const float pow2 = ldexpf(1.f, shift);
            uint32_t    ps[kNG][2][4];
#pragma unroll
            for(int u = 0; u < 2; ++u) { // tiles 2 u and 2 u + 1
                v4i sv[2][kNG];
#pragma unroll
                for(int i = 0; i < 2; ++i)
#pragma unroll
                    for(int g = 0; g < kNG; ++g)
                        sv[i][g] = *(const lds_v4i_t*)(uintptr_t)(
                            at + L::kCodes + L::kScales + (32 * u + 16 * i + 4 * kg) * kNG * 4
                            + g * 16);
#pragma unroll
                for(int j = 0; j < 4; ++j) {
                    const float p0 = p[8 * u + j], p1 = p[8 * u + 4 + j];
                    const float x0 = p0 * pow2, x1 = p1 * pow2;
#pragma unroll
                    for(int g = 0; g < kNG; ++g) {
                        const uint32_t w0 = (uint32_t)sv[0][(j * kNG + g) / 4][(j * kNG + g) % 4];
                        const uint32_t w1 = (uint32_t)sv[1][(j * kNG + g) / 4][(j * kNG + g) % 4];
                        osum[g]     = fmaf(p0, high_half(w0), fmaf(p1, high_half(w1), osum[g]));
                        ps[g][u][j] = scaled_pair(x0, w0, x1, w1);
                    }
                }
            }
            auto operand = [&](int g, int u) {
                return __builtin_bit_cast(
                    v8h, v4i{(int)ps[g][u][0], (int)ps[g][u][1], (int)ps[g][u][2], (int)ps[g][u][3]});
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
                const uint32_t f   = D == 128 ? tok / 4 % 4 : tok / 8 % 2;
                const v2i      w   = __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_v2i_t*)(uintptr_t)(
                    at + tok * (D / 2) + ((t / 2) ^ f) * 16 + t % 2 * 8));
#pragma unroll
                for(int u = 0; u < 2; ++u)
                    o[t] = mfma16(unpack((uint32_t)w[u]), operand(t * 16 / G, u), o[t]);
            }
        }
    }

    // ---- merge the waves ---------------------------------------------------------
    l                = column_sum(l);
    const float back = ldexpf(16.f, -shift);
#pragma unroll
    for(int g = 0; g < kNG; ++g) osum[g] = column_sum(osum[g]);
    __syncthreads(); // the ring is done with
    float* part = reinterpret_cast<float*>(lds);
    float* ml   = part + kAttWaves * kCols * D;
#pragma unroll
    for(int t = 0; t < kTiles; ++t) {
        const int g = t * 16 / G;
        v4f       r;
#pragma unroll
        for(int i = 0; i < 4; ++i) r[i] = fmaf(fmaf(total[g][i], -1.5f, o[t][i]), back, osum[g]);
        *reinterpret_cast<v4f*>(part + (wave * kCols + col) * D + 16 * t + 4 * kg) = r;
    }
    if(kg == 0) {
        ml[(wave * kCols + col) * 2]     = m * c2;
        ml[(wave * kCols + col) * 2 + 1] = l;
    }
    __syncthreads();
    for(uint32_t i = threadIdx.x; i < heads * D; i += kAttThreads) {
        const uint32_t h = i / D, ch = i % D;
        float          mm = -INFINITY;
#pragma unroll
        for(int w = 0; w < kAttWaves; ++w) mm = fmaxf(mm, ml[(w * kCols + h) * 2]);
        float sum = 0.f, ls = 0.f;
#pragma unroll
        for(int w = 0; w < kAttWaves; ++w) {
            const float lw = ml[(w * kCols + h) * 2 + 1];
            if(lw == 0.f) continue; // no token seen: its maximum may be -inf
            const float f = __builtin_amdgcn_exp2f(ml[(w * kCols + h) * 2] - mm);
            sum           = fmaf(f, part[(w * kCols + h) * D + ch], sum);
            ls            = fmaf(f, lw, ls);
        }
        if(pieces.count == 1)
            a.out[(size_t)seq * a.ldo + (size_t)(head0 + h) * D + ch]
                = float_to_half_bits(ls != 0.f ? sum / ls : 0.f);
        else {
            const size_t at         = ((size_t)seq * a.heads + head0 + h) * pieces.count + blockIdx.z;
            pieces.o[at * D + ch] = sum;
            if(ch == 0) {
                pieces.ml[at * 2]     = mm;
                pieces.ml[at * 2 + 1] = ls;
            }
        }
    }
}

template <int D, int G>
__global__ void __launch_bounds__(kAttThreads, 2)
    attention_kv4_kernel(CacheView c, AttentionKv4Args a, Pieces pieces, uint32_t pages)
{
    __shared__ alignas(16) uint8_t lds[KvLds<D, G>::kBytes];
    __shared__ int32_t             page_of[kSegment / 16];
    attention_kv4_piece<D, G>(c, a, pieces, pages, lds, page_of);
}

// Joins the pieces of one (sequence, head): their factors first, then the threads of
// each channel take every kJoin-th piece, and add up in a fixed order.
constexpr int kJoinThreads = 512, kJoinPieces = 256; // pieces whose factors lie in LDS at a time

template <int D>
__global__ void __launch_bounds__(kJoinThreads)
    attention_kv4_join_kernel(CacheView c, AttentionKv4Args a, Pieces pieces)
{
    constexpr int    kJoin = kJoinThreads / D;
    __shared__ float factor[kJoinPieces];
    __shared__ float part[kJoin][D + 1];
    const uint32_t   head = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x;
    const uint32_t   ch = tid % D, way = tid / D;
    const uint32_t   most = a.table_cols * c.page_size;
    const uint32_t   len  = (uint32_t)max(0, (int)min((int64_t)a.lens[seq], (int64_t)most));
    const uint32_t   n    = (len + pieces.tokens - 1) / pieces.tokens;
    const size_t     at   = ((size_t)seq * a.heads + head) * pieces.count;
    const float*     ml   = pieces.ml + at * 2;
    float            m    = -INFINITY; // of all pieces, in every wave
    for(uint32_t i = tid % kWave; i < n; i += kWave) m = fmaxf(m, ml[i * 2]);
    m         = wave_max(m);
    float sum = 0.f, l = 0.f;
    for(uint32_t i0 = 0; i0 < n; i0 += kJoinPieces) {
        const uint32_t here = min(n - i0, (uint32_t)kJoinPieces);
        __syncthreads();
        if(tid < here) {
            const float li = ml[(i0 + tid) * 2 + 1]; // 0: no token seen, its maximum may be -inf
            factor[tid]    = li != 0.f ? __builtin_amdgcn_exp2f(ml[(i0 + tid) * 2] - m) : 0.f;
        }
        __syncthreads();
#pragma unroll 8
        for(uint32_t i = way; i < here; i += kJoin) {
            const float f = factor[i];
            sum           = fmaf(f, pieces.o[(at + i0 + i) * D + ch], sum);
            l             = fmaf(f, ml[(i0 + i) * 2 + 1], l);
        }
    }
    part[way][ch] = sum;
    if(ch == 0) part[way][D] = l;
    __syncthreads();
    if(way != 0) return;
    for(int w = 1; w < kJoin; ++w) sum += part[w][ch];
    l = 0.f;
    for(int w = 0; w < kJoin; ++w) l += part[w][D];
    a.out[(size_t)seq * a.ldo + (size_t)head * D + ch] = float_to_half_bits(l != 0.f ? sum / l : 0.f);
}

// Pieces of equal size, as many as leave every one enough to do and fill the chip
// when every sequence is as long as its table.
constexpr uint32_t kPieceLeast = 256, kPieceBlocks = 1024;

uint32_t piece_tokens(uint32_t seqs, uint32_t heads, uint32_t kv_heads, uint32_t max_len)
{
    const uint32_t per    = heads / kv_heads;
    const uint64_t blocks = (uint64_t)seqs * kv_heads * ((per + kCols - 1) / kCols);
    const uint64_t t      = (blocks * max_len + kPieceBlocks - 1) / kPieceBlocks;
    return (uint32_t)std::min<uint64_t>((std::max<uint64_t>(t, 1) + kPieceLeast - 1) / kPieceLeast * kPieceLeast, 0x7FFFFF00u);
}

uint32_t piece_count(uint32_t tokens, uint32_t max_len)
{
    return std::max(1u, (uint32_t)(((uint64_t)max_len + tokens - 1) / tokens));
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
    const uint32_t n = piece_count(piece_tokens(seqs, heads, kv_heads, max_len), max_len);
    return n == 1 ? 0 : (size_t)seqs * heads * n * (dim + 2) * 4;
}

hipError_t launch_attention_kv4(const w8a8_kv4_cache& c, const AttentionKv4Args& a,
                                hipStream_t stream)
{
    const uint32_t max_len = a.table_cols * c.page_size;
    Pieces         pieces{1, 0, nullptr, nullptr};
    const size_t   need
        = attention_kv4_workspace_bytes(a.seqs, a.heads, c.kv_heads, c.head_dim, max_len);
    if(need != 0 && a.ws_bytes >= need) {
        pieces.tokens = piece_tokens(a.seqs, a.heads, c.kv_heads, max_len);
        pieces.count  = piece_count(pieces.tokens, max_len);
        pieces.o      = static_cast<float*>(a.ws);
        pieces.ml     = pieces.o + (size_t)a.seqs * a.heads * pieces.count * c.head_dim;
    }
    const uint32_t per = a.heads / c.kv_heads;
    const dim3     grid(c.kv_heads * ((per + kCols - 1) / kCols), a.seqs, pieces.count);
    with_widths(c, [&](auto d, auto g) {
        attention_kv4_kernel<d(), g()>
            <<<grid, kAttThreads, 0, stream>>>(view(c), a, pieces, c.pages);
        if(pieces.count > 1)
            attention_kv4_join_kernel<d()>
                <<<dim3(a.heads, a.seqs), kJoinThreads, 0, stream>>>(view(c), a, pieces);
    });
    return hipGetLastError();
}

} // namespace w8a8
