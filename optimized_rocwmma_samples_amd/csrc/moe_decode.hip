// moe_decode.hip -- the expert layer of the few tokens of a decode step for
// gfx950, in two launches (the chain of moe.hip takes nine):
//   gate_up_kernel  routing, the MoE quantizer, the gate_up products, SiLU(gate) * up
//   down_kernel     requantization, the down products, the weighted combine
// Both are streams of the active experts' weights, each byte read once; what the
// chain spreads over launches every block does again for itself, on a few KB from
// L2, while its first weights are in flight.
//   * v_mfma_i32_16x16x64_i8 with 16 weight rows as srcA (a lane loads 16
//     contiguous bytes of one row, a wave-load 64 bytes of 16 rows) and up to 16
//     quantized rows as srcB, read from LDS.  Sums are int32: exact, so the order
//     of the waves and blocks changes nothing.
//   * The 8 waves of a block split K; their int32 partials meet in LDS, one
//     barrier per 16 x 16 tile (the buffer alternates).
//   * The activations between the two kernels stay fp32 (a few hundred KB).  A row's
//     absmax comes from per-block maxima that the first kernel leaves beside them.
#include "moe_route.hpp"
#include "w8a8_device.hpp"
#include "w8a8_internal.hpp"

#include <algorithm>

namespace w8a8 {
namespace {

constexpr int      kThreads   = 512;
constexpr int      kWaves     = kThreads / kWave;
constexpr int      kRows      = W8A8_MOE_DECODE_MAX_TOKENS; // rows of an expert: one a token
constexpr int      kTile      = 16;                         // weight rows a tile
constexpr uint32_t kMaxExpert = 4096;
constexpr int      kWords     = kMaxExpert / 32;
constexpr int      kBufferFlags  = 0x00020000; // raw buffer, 32-bit data format
constexpr uint32_t kOob          = 0x80000000u;
constexpr int      kWeightPolicy = 2; // non-temporal: every weight byte is read once

constexpr uint32_t kGateUpBlocks = 512;        // two blocks a CU
constexpr uint32_t kDownRows     = 96 * 1024;  // bytes of quantized rows a block of down_kernel holds
constexpr uint32_t kLdsBytes     = 160 * 1024; // of a CU

static_assert(kRows == 16, "the rows are the columns of one 16 x 16 tile");
static_assert(W8A8_MOE_DECODE_MAX_VALUES + kRows * 80 + 64 * kRows * 4 + 36 * 1024 <= kLdsBytes,
              "a block of gate_up_kernel holds every token's row");

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// A quantized row in LDS: whole 64-byte steps (zeros past the row) and 16 bytes that
// spread the rows over the banks.
__host__ __device__ constexpr uint32_t row_bytes(uint32_t n) { return (n + 63) / 64 * 64 + 16; }

// Workspace between the kernels.
struct Ws {
    float*   act;    // [pairs, inter]
    float*   top;    // [pairs, kGateUpBlocks]: max |act| over a block's columns
    int32_t* ids;    // [pairs]
    float*   weight; // [pairs]
};

Ws carve(const MoeDecodeArgs& a)
{
    uint8_t*     p = static_cast<uint8_t*>(a.ws);
    const size_t n = (size_t)a.tokens * a.topk;
    Ws           w;
    w.act = reinterpret_cast<float*>(p);
    p += up256(n * a.inter * 4);
    w.top = reinterpret_cast<float*>(p);
    p += up256(n * kGateUpBlocks * 4);
    w.ids = reinterpret_cast<int32_t*>(p);
    p += up256(n * 4);
    w.weight = reinterpret_cast<float*>(p);
    return w;
}

__device__ __forceinline__ uint32_t wave_sum_u32(uint32_t v)
{
#pragma unroll
    for(int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, kWave);
    return v;
}

// The set of experts that some token is routed to, as bits in LDS, and its order.
struct Active {
    const uint32_t* bits; // [kWords]
    int             lane;

    __device__ uint32_t count() const
    {
        return wave_sum_u32(__popc(bits[2 * lane]) + __popc(bits[2 * lane + 1]));
    }
    // Active experts below e.
    __device__ uint32_t rank(uint32_t e) const
    {
        uint32_t n = 0;
#pragma unroll
        for(int i = 0; i < 2; ++i) {
            const uint32_t w = 2 * lane + i, b = bits[w];
            n += w < e / 32 ? __popc(b) : w == e / 32 ? __popc(b & ((1u << (e % 32)) - 1)) : 0;
        }
        return wave_sum_u32(n);
    }
    // The i-th active expert, i < count().
    __device__ uint32_t expert(uint32_t i) const
    {
        const uint32_t w0 = bits[2 * lane], w1 = bits[2 * lane + 1];
        const uint32_t n = __popc(w0) + __popc(w1);
        uint32_t       s = n;
#pragma unroll
        for(int d = 1; d < kWave; d <<= 1) {
            const uint32_t o = __shfl_up(s, d, kWave);
            if(lane >= d) s += o;
        }
        const int f = __builtin_ctzll(__ballot(s > i));
        i -= __builtin_amdgcn_readlane(s, f) - __builtin_amdgcn_readlane(n, f);
        uint32_t w = __builtin_amdgcn_readlane(w0, f), at = 2 * f;
        if(i >= (uint32_t)__popc(w)) {
            i -= __popc(w);
            w = __builtin_amdgcn_readlane(w1, f);
            ++at;
        }
        for(; i > 0; --i) w &= w - 1;
        return at * 32 + __builtin_ctz(w);
    }
};

// The pairs of expert e in ascending order into list[0 .. count), by one wave.
__device__ __forceinline__ uint32_t pairs_of(const int32_t* ids, uint32_t pairs, int32_t e,
                                             int lane, int32_t* list)
{
    uint32_t n = 0;
    for(uint32_t p0 = 0; p0 < pairs; p0 += kWave) {
        const uint32_t p    = p0 + lane;
        const bool     mine = p < pairs && ids[p] == e;
        const uint64_t mask = __ballot(mine);
        const uint32_t at   = n + __popcll(mask & ((1ull << lane) - 1));
        if(mine && at < (uint32_t)kRows) list[at] = (int32_t)p;
        n += __popcll(mask);
    }
    return min(n, (uint32_t)kRows);
}

// The columns of all active experts' activations, in tiles of 16, are cut into one
// contiguous range per block of gate_up_kernel.
__device__ __forceinline__ uint32_t first_unit(uint32_t block, uint32_t units, uint32_t blocks)
{
    return (uint32_t)((uint64_t)block * units / blocks);
}

__device__ __forceinline__ uint32_t block_of(uint32_t unit, uint32_t units, uint32_t blocks)
{
    return (uint32_t)((((uint64_t)unit + 1) * blocks - 1) / units);
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t weight_rows(const int8_t* w, uint32_t k)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(w), 0, (int)(kTile * k),
                                             kBufferFlags);
}

__device__ __forceinline__ v4i load_weights(__amdgpu_buffer_rsrc_t r, uint32_t offset)
{
    return __builtin_bit_cast(v4i,
                              __builtin_amdgcn_raw_buffer_load_b128(r, offset, 0, kWeightPolicy));
}

__device__ __forceinline__ v4i mfma(v4i a, v4i b, v4i c)
{
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// A wave's share of a row of K: its steps of 64 among `steps`.
struct Share {
    uint32_t from, to;
    __device__ Share(uint32_t steps, uint32_t wave)
        : from(steps * wave / kWaves), to(steps * (wave + 1) / kWaves)
    {
    }
    __device__ uint32_t batches(uint32_t per) const { return max(1u, (to - from + per - 1) / per); }
};

// ---------------------------------------------------------------------------
// First kernel
// ---------------------------------------------------------------------------
constexpr int kGuSteps = 4; // steps a batch: 4 KB of gate rows and 4 KB of up rows a wave

struct GateUpLds {
    v4i      part[2][kWaves][2][kWave];
    float    amax[kRows][kWaves];
    float    scale[kRows];
    float    top[4][kRows];
    uint32_t bits[kWords];
    int32_t  list[kRows];
};

template <bool F16>
__device__ __forceinline__ void gate_up(const MoeDecodeArgs& a, const Ws& ws, GateUpLds& lds,
                                        uint8_t* dyn)
{
    const int      wave  = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int      lane  = threadIdx.x % kWave, col = lane % 16, kg = lane / 16;
    const uint32_t pairs = a.tokens * a.topk, tid = threadIdx.x;
    int32_t*       ids = reinterpret_cast<int32_t*>(dyn);
    int8_t*        q   = reinterpret_cast<int8_t*>(dyn + (pairs * 4 + 15) / 16 * 16);
    const uint32_t rb  = row_bytes(a.hidden);

    // ---- routing: a wave per token -----------------------------------------------
    if(tid < kWords) lds.bits[tid] = 0;
    for(uint32_t t = wave; t < a.tokens; t += kWaves)
        route_token(
            [&](uint32_t e) { return load_logit<F16>(a.logits, (size_t)t * a.experts + e); },
            a.experts, a.topk, lane, [&](uint32_t k, int id, float w) {
                if(lane == 0) {
                    ids[t * a.topk + k] = id;
                    if(blockIdx.x == 0) {
                        ws.ids[t * a.topk + k]    = id;
                        ws.weight[t * a.topk + k] = w;
                    }
                }
            });
    __syncthreads();
    for(uint32_t p = tid; p < pairs; p += kThreads)
        if(ids[p] >= 0) atomicOr(&lds.bits[ids[p] / 32], 1u << (ids[p] % 32));
    __syncthreads();
    const Active   active{lds.bits, lane};
    const uint32_t tiles = a.inter / kTile, units = active.count() * tiles;
    const uint32_t from  = first_unit(blockIdx.x, units, gridDim.x);
    const uint32_t to    = first_unit(blockIdx.x + 1, units, gridDim.x);

    const uint32_t steps = (a.hidden + 63) / 64;
    const Share    share(steps, wave);
    const uint32_t batches = share.batches(kGuSteps);

    for(uint32_t u0 = from; u0 < to;) { // one expert's part of the block's range
        const uint32_t ai = u0 / tiles, u1 = min(to, (ai + 1) * tiles);
        const uint32_t e = active.expert(ai);
        const size_t   rows0 = (size_t)e * 2 * a.inter;

        v4i  ring[2][2][kGuSteps];
        auto load = [&](int slot, uint32_t at) { // batch `at` of the range, for this wave
            const uint32_t j0 = (u0 + at / batches - ai * tiles) * kTile;
            const uint32_t s0 = share.from + at % batches * kGuSteps;
            const __amdgpu_buffer_rsrc_t rg = weight_rows(a.wgu + (rows0 + j0) * a.hidden, a.hidden);
            const __amdgpu_buffer_rsrc_t ru
                = weight_rows(a.wgu + (rows0 + a.inter + j0) * a.hidden, a.hidden);
#pragma unroll
            for(int i = 0; i < kGuSteps; ++i) {
                const uint32_t off
                    = s0 + i < share.to ? col * a.hidden + (s0 + i) * 64 + kg * 16 : kOob;
                ring[slot][0][i] = load_weights(rg, off);
                ring[slot][1][i] = load_weights(ru, off);
            }
        };
        const uint32_t total = (u1 - u0) * batches;
        load(0, 0);

        // ---- the expert's rows, quantized into LDS ------------------------------
        __syncthreads(); // the rows and the list of the expert before are done with
        const uint32_t rows = pairs_of(ids, pairs, (int32_t)e, lane, lds.list);
        const float*   s    = a.s + (size_t)e * a.hidden;
        for(uint32_t r = 0; r < rows; ++r) {
            const uint16_t* x = a.x + (size_t)(lds.list[r] / a.topk) * a.ldx;
            float           m = 0.f;
            for(uint32_t k = tid * 8; k < a.hidden; k += kThreads * 8) {
                const v4i h  = *reinterpret_cast<const v4i*>(x + k);
                const v4f s0 = *reinterpret_cast<const v4f*>(s + k);
                const v4f s1 = *reinterpret_cast<const v4f*>(s + k + 4);
#pragma unroll
                for(int i = 0; i < 4; ++i) {
                    const float sa = i < 2 ? s0[2 * i] : s1[2 * i - 4];
                    const float sb = i < 2 ? s0[2 * i + 1] : s1[2 * i - 3];
                    m = fmaxf(m, fabsf(mul_h16_f32<false>((uint32_t)h[i], sa)));
                    m = fmaxf(m, fabsf(mul_h16_f32<true>((uint32_t)h[i], sb)));
                }
            }
            m = wave_max(m);
            if(lane == 0) lds.amax[r][wave] = m;
        }
        __syncthreads();
        for(uint32_t r = 0; r < rows; ++r) {
            float m = lds.amax[r][0];
#pragma unroll
            for(int w = 1; w < kWaves; ++w) m = fmaxf(m, lds.amax[r][w]);
            const float scale = m / a.qmax;
            const float inv   = scale > 0.f ? 1.f / scale : 0.f;
            if(tid == 0) lds.scale[r] = scale;
            const uint16_t* x = a.x + (size_t)(lds.list[r] / a.topk) * a.ldx;
            for(uint32_t k = tid * 8; k < rb - 16; k += kThreads * 8) {
                v2i w = {0, 0};
                if(k < a.hidden) {
                    const v4i h  = *reinterpret_cast<const v4i*>(x + k);
                    const v4f s0 = *reinterpret_cast<const v4f*>(s + k);
                    const v4f s1 = *reinterpret_cast<const v4f*>(s + k + 4);
                    float     f[8];
#pragma unroll
                    for(int i = 0; i < 4; ++i) {
                        const float sa = i < 2 ? s0[2 * i] : s1[2 * i - 4];
                        const float sb = i < 2 ? s0[2 * i + 1] : s1[2 * i - 3];
                        f[2 * i] = quant_f(mul_h16_f32<false>((uint32_t)h[i], sa), inv, a.qmax);
                        f[2 * i + 1] = quant_f(mul_h16_f32<true>((uint32_t)h[i], sb), inv, a.qmax);
                    }
                    w[0] = (int)cvt_pack4_i8(f[0], f[1], f[2], f[3]);
                    w[1] = (int)cvt_pack4_i8(f[4], f[5], f[6], f[7]);
                }
                *reinterpret_cast<v2i*>(q + r * rb + k) = w;
            }
        }
        __syncthreads();

        // ---- the products -------------------------------------------------------
        const int8_t* qrow = q + min((uint32_t)col, rows - 1) * rb + kg * 16;
        // the epilogue's place: waves 0..3, lane = (row lane / 4, column 4 wave + lane % 4)
        const uint32_t er = lane / 4, ej = 4 * (wave % 4) + lane % 4;
        const bool     epilogue = wave < 4 && er < rows;
        const int32_t  epair    = epilogue ? lds.list[er] : 0;
        const float    escale   = epilogue ? lds.scale[er] : 0.f;
        float          top = 0.f, sg = 0.f, su = 0.f, s2 = 1.f;
        v4i            acc[2] = {};
        auto process = [&](int slot, uint32_t at) {
            const uint32_t unit = u0 + at / batches, b = at % batches;
            const uint32_t j = (unit - ai * tiles) * kTile + ej;
            if(b == 0) {
                acc[0] = acc[1] = v4i{0, 0, 0, 0};
                if(epilogue) {
                    sg = a.sgu[rows0 + j];
                    su = a.sgu[rows0 + a.inter + j];
                    if(a.s2) s2 = a.s2[(size_t)e * a.inter + j];
                }
            }
#pragma unroll
            for(int i = 0; i < kGuSteps; ++i) {
                const uint32_t st = min(share.from + b * kGuSteps + i, steps - 1);
                const v4i      x  = *reinterpret_cast<const v4i*>(qrow + st * 64);
                acc[0]            = mfma(ring[slot][0][i], x, acc[0]);
                acc[1]            = mfma(ring[slot][1][i], x, acc[1]);
            }
            if(b + 1 < batches) return;
            v4i(*part)[2][kWave]  = lds.part[unit % 2];
            part[wave][0][lane] = acc[0];
            part[wave][1][lane] = acc[1];
            __syncthreads();
            if(!epilogue) return;
            int g = 0, u = 0;
#pragma unroll
            for(int w = 0; w < kWaves; ++w) {
                g += reinterpret_cast<const int*>(part[w][0])[(wave * 16 + er) * 4 + lane % 4];
                u += reinterpret_cast<const int*>(part[w][1])[(wave * 16 + er) * 4 + lane % 4];
            }
            const float h = silu_mul(((float)g * escale) * sg, ((float)u * escale) * su)
                            * s2;
            ws.act[(size_t)epair * a.inter + j] = h;
            top                                 = fmaxf(top, fabsf(h));
        };
        for(uint32_t at = 0; at < total; at += 2) {
            if(at + 1 < total) load(1, at + 1);
            process(0, at);
            if(at + 1 < total) {
                if(at + 2 < total) load(0, at + 2);
                process(1, at + 1);
            }
        }
        if(epilogue) {
            top = fmaxf(top, dpp_mov<kDppQuadXor1>(top));
            top = fmaxf(top, dpp_mov<kDppQuadXor2>(top));
            if(lane % 4 == 0) lds.top[wave][er] = top;
        }
        __syncthreads();
        if(tid < rows)
            ws.top[(size_t)lds.list[tid] * kGateUpBlocks + blockIdx.x] = fmaxf(
                fmaxf(lds.top[0][tid], lds.top[1][tid]), fmaxf(lds.top[2][tid], lds.top[3][tid]));
        u0 = u1;
    }
}

template <bool F16>
__global__ void __launch_bounds__(kThreads, 4) gate_up_kernel(MoeDecodeArgs a, Ws ws)
{
    extern __shared__ uint8_t dyn[];
    __shared__ GateUpLds      lds;
    gate_up<F16>(a, ws, lds, dyn);
}

// ---------------------------------------------------------------------------
// Second kernel: a block owns 16 output columns of all active experts.
// ---------------------------------------------------------------------------
constexpr int kDownSteps = 8; // steps a batch: 8 KB a wave

struct DownLds {
    v4i      part[2][kWaves][kWave];
    uint32_t bits[kWords];
    int32_t  list[2][kWaves][kRows];
};

// How the quantized rows lie in LDS: all pairs' whole rows at once (chunk = inter), or
// one expert's rows over `chunk` columns at a time.
struct DownPlan {
    uint32_t chunk;
    bool     all;
};

__device__ __forceinline__ void down(const MoeDecodeArgs& a, const Ws& ws, const DownPlan& plan,
                                     uint32_t gu_blocks, DownLds& lds, uint8_t* dyn)
{
    const int      wave  = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int      lane  = threadIdx.x % kWave, col = lane % 16, kg = lane / 16;
    const uint32_t pairs = a.tokens * a.topk, tid = threadIdx.x;
    const uint32_t up16  = (pairs * 4 + 15) / 16 * 16;
    int32_t*       ids   = reinterpret_cast<int32_t*>(dyn);
    float*         scale = reinterpret_cast<float*>(dyn + up16);
    float*         y     = reinterpret_cast<float*>(dyn + 2 * up16); // [pairs][16]
    int8_t*        q     = reinterpret_cast<int8_t*>(dyn + 2 * up16 + pairs * kTile * 4);
    const uint32_t j0 = blockIdx.x * kTile, rb = row_bytes(plan.chunk);

    if(tid < kWords) lds.bits[tid] = 0;
    for(uint32_t p = tid; p < pairs; p += kThreads) ids[p] = ws.ids[p];
    __syncthreads();
    for(uint32_t p = tid; p < pairs; p += kThreads)
        if(ids[p] >= 0) atomicOr(&lds.bits[ids[p] / 32], 1u << (ids[p] % 32));
    __syncthreads();
    const Active   active{lds.bits, lane};
    const uint32_t n = active.count(), tiles = a.inter / kTile, units = n * tiles;
    const uint32_t chunks = (a.inter + plan.chunk - 1) / plan.chunk;

    // ---- the stream of weights: (expert, chunk, batch), one batch ahead ------------
    struct Cursor {
        uint32_t ai, ci, b, e;
    };
    auto steps_of = [&](uint32_t ci) {
        return (min(plan.chunk, a.inter - ci * plan.chunk) + 63) / 64;
    };
    auto advance = [&](Cursor& c) {
        if(++c.b < Share(steps_of(c.ci), wave).batches(kDownSteps)) return;
        c.b = 0;
        if(++c.ci < chunks) return;
        c.ci = 0;
        if(++c.ai < n) c.e = active.expert(c.ai);
    };
    v4i  ring[2][kDownSteps];
    auto load = [&](int slot, const Cursor& c) {
        const Share                  share(steps_of(c.ci), wave);
        const __amdgpu_buffer_rsrc_t r
            = weight_rows(a.wd + ((size_t)c.e * a.hidden + j0) * a.inter, a.inter);
        const uint32_t s0 = share.from + c.b * kDownSteps;
#pragma unroll
        for(int i = 0; i < kDownSteps; ++i)
            ring[slot][i] = load_weights(r, s0 + i < share.to ? col * a.inter + c.ci * plan.chunk
                                                                    + (s0 + i) * 64 + kg * 16
                                                              : kOob);
    };
    Cursor now{0, 0, 0, n > 0 ? active.expert(0) : 0}, ahead = now;
    if(n > 0) {
        load(0, ahead);
        advance(ahead);
    }

    // ---- the pairs' scales, from the maxima that the first kernel's blocks left -----
    for(uint32_t p = wave; p < pairs; p += kWaves) {
        float m = 0.f;
        if(ids[p] >= 0) {
            const uint32_t ai = active.rank(ids[p]);
            const uint32_t b0 = block_of(ai * tiles, units, gu_blocks);
            const uint32_t b1 = block_of(ai * tiles + tiles - 1, units, gu_blocks);
            for(uint32_t b = b0 + lane; b <= b1; b += kWave)
                if(first_unit(b, units, gu_blocks) < first_unit(b + 1, units, gu_blocks))
                    m = fmaxf(m, ws.top[(size_t)p * kGateUpBlocks + b]); // it had work
            m = wave_max(m);
        }
        if(lane == 0) scale[p] = m / a.qmax;
    }
    __syncthreads();

    // 16 columns a thread from k0 + 16 i on of one pair's row, to LDS row `row`
    auto quantize = [&](uint32_t p, uint32_t row, uint32_t k0, uint32_t i) {
        const float  inv = scale[p] > 0.f ? 1.f / scale[p] : 0.f;
        const float* h   = ws.act + (size_t)p * a.inter + k0 + 16 * i;
        v4i          w   = {0, 0, 0, 0};
        if(k0 + 16 * i < a.inter) {
#pragma unroll
            for(int c = 0; c < 4; ++c) {
                const v4f f = *reinterpret_cast<const v4f*>(h + 4 * c);
                w[c] = (int)cvt_pack4_i8(quant_f(f[0], inv, a.qmax), quant_f(f[1], inv, a.qmax),
                                         quant_f(f[2], inv, a.qmax), quant_f(f[3], inv, a.qmax));
            }
        }
        *reinterpret_cast<v4i*>(q + row * rb + 16 * i) = w;
    };
    const uint32_t per_row = (rb - 16) / 16;
    if(plan.all) {
        for(uint32_t i = tid; i < pairs * per_row; i += kThreads)
            if(ids[i / per_row] >= 0) quantize(i / per_row, i / per_row, 0, i % per_row);
        __syncthreads();
    }

    v4i           acc  = {};
    uint32_t      rows = 0;
    const int8_t* qrow = q;
    float         sd   = 0.f;
    // the epilogue's place: waves 0..3, lane = (row lane / 4, column 4 wave + lane % 4)
    const uint32_t er = lane / 4, ej = 4 * (wave % 4) + lane % 4;
    auto process = [&](int slot) {
        if(now.b == 0) {
            if(now.ci == 0) { // another expert
                acc  = v4i{0, 0, 0, 0};
                rows = pairs_of(ids, pairs, (int32_t)now.e, lane, lds.list[now.ai % 2][wave]);
                sd   = a.sd[(size_t)now.e * a.hidden + j0 + ej];
            }
            const int32_t* list = lds.list[now.ai % 2][wave];
            const uint32_t mine = min((uint32_t)col, rows - 1);
            if(!plan.all) {
                __syncthreads(); // the rows before are done with
                for(uint32_t i = tid; i < rows * per_row; i += kThreads)
                    quantize(list[i / per_row], i / per_row, now.ci * plan.chunk, i % per_row);
                __syncthreads();
            }
            qrow = q + (plan.all ? list[mine] : mine) * rb + kg * 16;
        }
        const uint32_t steps = steps_of(now.ci);
        const Share    share(steps, wave);
#pragma unroll
        for(int i = 0; i < kDownSteps; ++i) {
            const uint32_t st = min(share.from + now.b * kDownSteps + i, steps - 1);
            acc = mfma(ring[slot][i], *reinterpret_cast<const v4i*>(qrow + st * 64), acc);
        }
        const Cursor done = now;
        advance(now);
        if(now.ai == done.ai) return;
        v4i(*part)[kWave] = lds.part[done.ai % 2];
        part[wave][lane]  = acc;
        __syncthreads();
        if(wave >= 4 || er >= rows) return;
        const int32_t p   = lds.list[done.ai % 2][wave][er];
        int           sum = 0;
#pragma unroll
        for(int w = 0; w < kWaves; ++w)
            sum += reinterpret_cast<const int*>(part[w])[(wave * 16 + er) * 4 + lane % 4];
        y[p * kTile + ej] = ((float)sum * scale[p]) * sd;
    };
    while(now.ai < n) {
        if(ahead.ai < n) {
            load(1, ahead);
            advance(ahead);
        }
        process(0);
        if(now.ai >= n) break;
        if(ahead.ai < n) {
            load(0, ahead);
            advance(ahead);
        }
        process(1);
    }
    __syncthreads();

    // ---- the weighted sum over a token's slots -------------------------------------
    for(uint32_t i = tid; i < a.tokens * kTile; i += kThreads) {
        const uint32_t t = i / kTile, j = i % kTile;
        float          out = 0.f;
        for(uint32_t s = 0; s < a.topk; ++s) {
            const uint32_t p = t * a.topk + s;
            if(ids[p] >= 0) out = fmaf(ws.weight[p], y[p * kTile + j], out);
        }
        a.out[(size_t)t * a.ldo + j0 + j] = float_to_half_bits(out);
    }
}

__global__ void __launch_bounds__(kThreads, 4)
    down_kernel(MoeDecodeArgs a, Ws ws, DownPlan plan, uint32_t gu_blocks)
{
    extern __shared__ uint8_t dyn[];
    __shared__ DownLds        lds;
    down(a, ws, plan, gu_blocks, lds, dyn);
}

} // namespace

size_t moe_ffn_decode_workspace_bytes(uint32_t tokens, uint32_t topk, uint32_t hidden, uint32_t inter)
{
    const size_t n = (size_t)tokens * topk;
    return up256(n * inter * 4) + up256(n * kGateUpBlocks * 4) + 2 * up256(n * 4);
}

namespace {
template <class K>
void allow_lds(K kernel, uint32_t bytes)
{
    if(bytes > 32 * 1024) // beside the static part
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                  hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}
} // namespace

hipError_t launch_moe_ffn_decode(const MoeDecodeArgs& a, bool f16, hipStream_t stream)
{
    const Ws       ws    = carve(a);
    const uint32_t pairs = a.tokens * a.topk, up16 = (pairs * 4 + 15) / 16 * 16;
    const uint32_t used   = std::min(pairs, a.experts);
    const uint32_t blocks = std::min(kGateUpBlocks, used * (a.inter / kTile));
    const uint32_t gu_lds = up16 + a.tokens * row_bytes(a.hidden);
    const auto     gu     = f16 ? gate_up_kernel<true> : gate_up_kernel<false>;
    allow_lds(gu, gu_lds);
    gu<<<blocks, kThreads, gu_lds, stream>>>(a, ws);
    hipError_t e = hipGetLastError();
    if(e != hipSuccess) return e;

    const uint32_t fixed = 2 * up16 + pairs * kTile * 4;
    const uint32_t rows
        = std::min<uint32_t>(kDownRows, kLdsBytes - (uint32_t)sizeof(DownLds) - fixed);
    DownPlan plan{a.inter, true};
    if((uint64_t)pairs * row_bytes(a.inter) > rows) {
        plan.all   = false;
        plan.chunk = std::min(a.inter, (rows / a.tokens - 16) / 512 * 512);
    }
    const uint32_t down_lds = fixed + (plan.all ? pairs : a.tokens) * row_bytes(plan.chunk);
    allow_lds(down_kernel, down_lds);
    down_kernel<<<a.hidden / kTile, kThreads, down_lds, stream>>>(a, ws, plan, blocks);
    return hipGetLastError();
}

} // namespace w8a8
