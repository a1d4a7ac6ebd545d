// moe_decode.hip -- the expert layer of the few tokens of a decode step for
// gfx950, in three launches (the chain of moe.hip takes nine):
//   gate_up_kernel  routing, the MoE quantizer, the gate_up products, SiLU(gate) * up
//   requant_kernel  the activations in 8 bits
//   down_kernel     the down products, the weighted combine
// The first and the last are streams of the active experts' weights, each byte read once
// (8 experts of 4096 x 14336: one token 75 us, 4.7 TB/s; 16 tokens 256 us, 5.5 TB/s).
// Routing and quantization, which the chain has launches for, every block of the first
// does again for itself, on a few KB from L2.  What is left above the bytes is that
// start, a chain of short dependent steps, the second launch (4.7 us), and weight loads
// that are not ahead: they are issued under conditions (the run's end), and where the
// paths meet the compiler waits for all of them, so that every batch ends on an empty
// queue and other waves alone fill the time.
//   * v_mfma_i32_16x16x64_i8 with 16 weight rows as srcA (a lane loads 16
//     contiguous bytes of one row, a wave-load 64 bytes of 16 rows) and up to 16
//     quantized rows as srcB, read from LDS or L2.
//   * A block's steps along K, over all its tiles or experts, are cut into 8 equal
//     runs, one per wave; a wave adds its int32 sums to LDS where it leaves a tile.
//     Integer sums are exact, so no order changes anything, and the stream has no
//     barrier in it (a barrier per tile cost 1.5 us each: 5 tokens of 64 experts of
//     2048 x 1408 106 us, 51 now).
//   * The activations between the kernels stay fp32 until they are quantized (a few
//     hundred KB).  A row's absmax comes from per-block maxima beside them.
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
constexpr uint32_t kMaxTopk   = 32;
constexpr int      kBufferFlags  = 0x00020000; // raw buffer, 32-bit data format
constexpr uint32_t kOob          = 0x80000000u;
// Default cache policy, although every byte is read once: a wave-load takes half of each
// 128-byte line, and non-temporal lines were gone before the other half's load (64
// experts of 7168 x 2048, 16 tokens, 539 us against 487).
constexpr int kWeightPolicy = 0;

constexpr uint32_t kCus          = 256;
constexpr uint32_t kGateUpBlocks = 2 * kCus;
constexpr uint32_t kLdsBytes     = 160 * 1024; // of a CU

static_assert(kRows == 16, "the rows are the columns of one 16 x 16 tile");

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// A quantized row in LDS: whole 64-byte steps (zeros past the row) and 16 bytes that
// spread the rows over the banks.
__host__ __device__ constexpr uint32_t row_bytes(uint32_t n) { return (n + 63) / 64 * 64 + 16; }

// Workspace between the kernels.
struct Ws {
    float*   act;    // [pairs, inter]
    float*   top;    // [kGateUpBlocks, pairs]: max |act| over a block's columns
    uint8_t* lists;  // as in LDS
    int32_t* active; // experts in them
    float*   weight; // [pairs]
    float*   scale;  // [pairs]: of the quantized activations
    int8_t*  q;      // [pairs, inter]: those
};

// The active experts (those some token is routed to) in ascending order, each with
// its pairs (token * topk + slot) in ascending order.  In LDS, sized by the pairs.
struct Lists {
    int32_t*  ids;    // [pairs] a pair's expert, or -1
    int32_t*  expert; // [active]
    int32_t*  count;  // [active] pairs
    uint16_t* pair;   // [active][16]

    __host__ __device__ static constexpr uint32_t up16(uint32_t pairs)
    {
        return (pairs * 4 + 15) / 16 * 16;
    }
    __host__ __device__ static constexpr uint32_t bytes(uint32_t pairs)
    {
        return 3 * up16(pairs) + (pairs * kRows * 2 + 15) / 16 * 16;
    }
    __device__ Lists(uint8_t* lds, uint32_t pairs)
    {
        const uint32_t n = up16(pairs);
        ids    = reinterpret_cast<int32_t*>(lds);
        expert = reinterpret_cast<int32_t*>(lds + n);
        count  = reinterpret_cast<int32_t*>(lds + 2 * n);
        pair   = reinterpret_cast<uint16_t*>(lds + 3 * n);
    }
    // From the ids in LDS, by all threads, with `bits` [kWords] and `active` zeroed;
    // barriers before and after.
    __device__ void build(uint32_t pairs, uint32_t* bits, uint32_t* active)
    {
        for(uint32_t p = threadIdx.x; p < pairs; p += kThreads) {
            count[p] = 0;
            if(ids[p] >= 0) atomicOr(&bits[ids[p] / 32], 1u << (ids[p] % 32));
        }
        __syncthreads();
        for(uint32_t p = threadIdx.x; p < pairs; p += kThreads) {
            const int32_t e = ids[p];
            if(e < 0) continue;
            uint32_t i = __popc(bits[e / 32] & ((1u << (e % 32)) - 1)), at = 0;
            for(int32_t w = 0; w < e / 32; ++w) i += __popc(bits[w]);
#pragma unroll 4
            for(uint32_t o = 0; o < p; ++o) at += ids[o] == e;
            expert[i] = e;
            if(at < (uint32_t)kRows) pair[i * kRows + at] = (uint16_t)p;
            if(at == 0) atomicAdd(active, 1u);
            atomicAdd(&count[i], 1);
        }
        __syncthreads();
    }
    __device__ uint32_t expert_at(uint32_t i) const
    {
        return (uint32_t)__builtin_amdgcn_readfirstlane(expert[i]);
    }
    __device__ uint32_t rows(uint32_t i) const
    {
        return (uint32_t)__builtin_amdgcn_readfirstlane(min(count[i], kRows));
    }
};

Ws carve(const MoeDecodeArgs& a)
{
    uint8_t*       p = static_cast<uint8_t*>(a.ws);
    const uint32_t n = a.tokens * a.topk;
    auto           take = [&](size_t bytes) {
        uint8_t* at = p;
        p += up256(bytes);
        return at;
    };
    Ws w;
    w.act    = reinterpret_cast<float*>(take((size_t)n * a.inter * 4));
    w.top    = reinterpret_cast<float*>(take((size_t)n * kGateUpBlocks * 4));
    w.lists  = take(Lists::bytes(n));
    w.active = reinterpret_cast<int32_t*>(take(4));
    w.weight = reinterpret_cast<float*>(take(n * 4));
    w.scale  = reinterpret_cast<float*>(take(n * 4));
    w.q      = reinterpret_cast<int8_t*>(take((size_t)n * a.inter));
    return w;
}

// The columns of all active experts' activations, in tiles of 16, are cut into one
// contiguous range per block of gate_up_kernel.
__device__ __forceinline__ uint32_t first_unit(uint32_t block, uint32_t units, uint32_t blocks)
{
    return block * units / blocks; // units <= 512 * 2048, blocks <= 512
}

// Hardware gives blocks to the 8 XCDs in turn; an index such that each XCD has a
// contiguous range of them.
__device__ __forceinline__ uint32_t xcd_range(uint32_t block, uint32_t blocks)
{
    const uint32_t x = block % 8, r = blocks % 8;
    return x * (blocks / 8) + min(x, r) + block / 8;
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

// A wave's run of `total` batches, and a place in it: batch b of item `item`, `per`
// batches an item.
struct Run {
    uint32_t from, to;
    __device__ Run(uint32_t total, uint32_t wave)
        : from(total * wave / kWaves), to(total * (wave + 1) / kWaves)
    {
    }
};

struct Cursor {
    uint32_t item, b;
    __device__ Cursor(uint32_t at, uint32_t per) : item(at / per), b(at % per) {}
    __device__ void advance(uint32_t per)
    {
        if(++b == per) {
            b = 0;
            ++item;
        }
    }
};

// ---------------------------------------------------------------------------
// First kernel: a block owns a range of 16-column tiles of the activations.
// ---------------------------------------------------------------------------
constexpr int      kGuSteps = 2; // steps a batch: 2 KB of gate rows and 2 KB of up rows a wave

// Sums of a tile in LDS: [gate, up][row][column].  As many tiles at a time as `group`.
typedef int32_t TileSums[2][kRows][kTile];

struct GateUpLds {
    float    amax[kRows][kWaves];
    float    scale[kRows];
    uint32_t bits[kWords];
    uint32_t active;
};

static_assert(W8A8_MOE_DECODE_MAX_VALUES + kRows * 80 + Lists::bytes(kRows * kMaxTopk)
                      + Lists::up16(kRows * kMaxTopk) + sizeof(GateUpLds) + 4 * sizeof(TileSums)
                  <= kLdsBytes,
              "a block of gate_up_kernel holds every token's row");

// RING: batches in registers, loaded up to RING - 1 ahead (see above for the waits).
template <bool F16, int RING>
__device__ __forceinline__ void gate_up(const MoeDecodeArgs& a, const Ws& ws, uint32_t group,
                                        GateUpLds& lds, uint8_t* dyn)
{
    const int      wave  = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int      lane  = threadIdx.x % kWave, col = lane % 16, kg = lane / 16;
    const uint32_t pairs = a.tokens * a.topk, tid = threadIdx.x;
    Lists          lists(dyn, pairs);
    uint32_t*      top  = reinterpret_cast<uint32_t*>(dyn + Lists::bytes(pairs)); // [pairs]
    TileSums*      sums
        = reinterpret_cast<TileSums*>(dyn + Lists::bytes(pairs) + Lists::up16(pairs));
    int8_t*        q    = reinterpret_cast<int8_t*>(sums + group);
    const uint32_t rb   = row_bytes(a.hidden);

    // ---- routing: a wave per token -----------------------------------------------
    if(tid < kWords) lds.bits[tid] = 0;
    if(tid == 0) lds.active = 0;
    for(uint32_t p = tid; p < pairs; p += kThreads) top[p] = 0; // float bits, >= 0
    for(uint32_t t = wave; t < a.tokens; t += kWaves)
        route_token(
            [&](uint32_t e) { return load_logit<F16>(a.logits, (size_t)t * a.experts + e); },
            a.experts, a.topk, lane, [&](uint32_t k, int id, float w) {
                if(lane == 0) {
                    lists.ids[t * a.topk + k] = id;
                    if(blockIdx.x == 0) ws.weight[t * a.topk + k] = w;
                }
            });
    __syncthreads();
    lists.build(pairs, lds.bits, &lds.active);
    if(blockIdx.x == 0) { // for the down kernel
        for(uint32_t i = tid; i < Lists::bytes(pairs) / 16; i += kThreads)
            reinterpret_cast<v4i*>(ws.lists)[i] = reinterpret_cast<const v4i*>(dyn)[i];
        if(tid == 0) *ws.active = (int32_t)lds.active;
    }
    const uint32_t tiles = a.inter / kTile, units = lds.active * tiles;
    // neighbouring ranges to one XCD: where every other block has a tile more, each XCD
    // gets as many of both (8 experts of 4096 x 14336, one token: 448 and 448 tiles at
    // 3.5 a block; round robin gave half the XCDs a third more, 48 us against 38)
    const uint32_t range = xcd_range(blockIdx.x, gridDim.x);
    const uint32_t from  = first_unit(range, units, gridDim.x);
    const uint32_t to    = first_unit(range + 1, units, gridDim.x);
    const uint32_t steps = (a.hidden + 63) / 64, per = (steps + kGuSteps - 1) / kGuSteps;

    uint32_t held = ~0u; // the expert whose rows are in LDS
    for(uint32_t u0 = from; u0 < to;) { // tiles u0 .. u1 of one expert
        const uint32_t ai = u0 / tiles, u1 = min(min(to, (ai + 1) * tiles), u0 + group);
        const uint32_t e = lists.expert_at(ai), rows = lists.rows(ai);
        const size_t   row0 = (size_t)e * 2 * a.inter + (u0 - ai * tiles) * kTile;
        const uint16_t* list = lists.pair + ai * kRows;

        // ---- the first of the expert's rows, ahead of the weights ----------------
        const float* s     = a.s + (size_t)e * a.hidden;
        const bool   fresh = held != e;
        auto         row_x = [&](uint32_t r) {
            return a.x + (size_t)(list[min(r, rows - 1)] / a.topk) * a.ldx;
        };
        v4i h[4] = {};
        v4f s0 = {}, s1 = {};
        auto fetch = [&](uint32_t r0, uint32_t k) {
            if(k < a.hidden) {
                s0 = *reinterpret_cast<const v4f*>(s + k);
                s1 = *reinterpret_cast<const v4f*>(s + k + 4);
#pragma unroll
                for(int i = 0; i < 4; ++i) h[i] = *reinterpret_cast<const v4i*>(row_x(r0 + i) + k);
            } else {
                s0 = s1 = v4f{0, 0, 0, 0};
#pragma unroll
                for(int i = 0; i < 4; ++i) h[i] = v4i{0, 0, 0, 0};
            }
        };
        if(fresh) fetch(0, tid * 8);

        // ---- the stream of weights ----------------------------------------------
        const Run run((u1 - u0) * per, wave);
        v4i       ring[RING][2][kGuSteps];
        Cursor    ahead(run.from, per), now = ahead;
        uint32_t  at   = run.from;
        auto      load = [&](int slot) {
            const size_t                 row = row0 + ahead.item * kTile;
            const __amdgpu_buffer_rsrc_t rg = weight_rows(a.wgu + row * a.hidden, a.hidden);
            const __amdgpu_buffer_rsrc_t ru
                = weight_rows(a.wgu + (row + a.inter) * a.hidden, a.hidden);
#pragma unroll
            for(int i = 0; i < kGuSteps; ++i) {
                const uint32_t st  = ahead.b * kGuSteps + i;
                const uint32_t off = st < steps ? col * a.hidden + st * 64 + kg * 16 : kOob;
                ring[slot][0][i]   = load_weights(rg, off);
                ring[slot][1][i]   = load_weights(ru, off);
            }
            ahead.advance(per);
            ++at;
        };
#pragma unroll
        for(int i = 0; i < RING - 1; ++i)
            if(at < run.to) load(i);

        __syncthreads(); // the sums and rows before are done with
        for(uint32_t i = tid; i < (u1 - u0) * sizeof(TileSums) / 16; i += kThreads)
            reinterpret_cast<v4i*>(sums)[i] = v4i{0, 0, 0, 0};
        // ---- the expert's rows, quantized into LDS: four rows at a time, so that
        // their loads overlap ------------------------------------------------------
        if(fresh) {
            auto product = [&](int i, int c) {
                const float f = c < 4 ? s0[c] : s1[c - 4];
                return c % 2 ? mul_h16_f32<true>((uint32_t)h[i][c / 2], f)
                             : mul_h16_f32<false>((uint32_t)h[i][c / 2], f);
            };
            const bool once = rows <= 4 && rb - 16 <= kThreads * 8; // they stay in registers
            for(uint32_t r0 = 0; r0 < rows; r0 += 4) {
                float m[4] = {};
                for(uint32_t k = tid * 8; k < rb - 16; k += kThreads * 8) {
                    if(r0 > 0 || k != tid * 8) fetch(r0, k);
#pragma unroll
                    for(int i = 0; i < 4; ++i)
#pragma unroll
                        for(int c = 0; c < 8; ++c) m[i] = fmaxf(m[i], fabsf(product(i, c)));
                }
#pragma unroll
                for(int i = 0; i < 4; ++i) {
                    m[i] = wave_max(m[i]);
                    if(lane == 0) lds.amax[r0 + i][wave] = m[i];
                }
            }
            __syncthreads();
            for(uint32_t r0 = 0; r0 < rows; r0 += 4) {
                float inv[4];
#pragma unroll
                for(int i = 0; i < 4; ++i) {
                    float m = lds.amax[r0 + i][0];
#pragma unroll
                    for(int w = 1; w < kWaves; ++w) m = fmaxf(m, lds.amax[r0 + i][w]);
                    const float scale = m / a.qmax;
                    inv[i]            = scale > 0.f ? 1.f / scale : 0.f;
                    if(tid == 0) lds.scale[r0 + i] = scale;
                }
                for(uint32_t k = tid * 8; k < rb - 16; k += kThreads * 8) {
                    if(!once) fetch(r0, k);
#pragma unroll
                    for(int i = 0; i < 4; ++i) {
                        float g[8];
#pragma unroll
                        for(int c = 0; c < 8; ++c) g[c] = quant_f(product(i, c), inv[i], a.qmax);
                        const v2i w = {(int)cvt_pack4_i8(g[0], g[1], g[2], g[3]),
                                       (int)cvt_pack4_i8(g[4], g[5], g[6], g[7])};
                        if(r0 + i < rows) *reinterpret_cast<v2i*>(q + (r0 + i) * rb + k) = w;
                    }
                }
            }
            held = e;
        }
        __syncthreads();

        // ---- the products -------------------------------------------------------
        const int8_t* qrow = q + min((uint32_t)col, rows - 1) * rb + kg * 16;
        v4i           acc[2] = {};
        for(uint32_t done = run.from; done < run.to;) {
#pragma unroll
            for(int slot = 0; slot < RING; ++slot) {
                if(at < run.to) load((slot + RING - 1) % RING);
                if(done < run.to) {
#pragma unroll
                    for(int i = 0; i < kGuSteps; ++i) {
                        const uint32_t st = min(now.b * kGuSteps + i, steps - 1);
                        const v4i      x  = *reinterpret_cast<const v4i*>(qrow + st * 64);
                        acc[0]            = mfma(ring[slot][0][i], x, acc[0]);
                        acc[1]            = mfma(ring[slot][1][i], x, acc[1]);
                    }
                    ++done;
                    if(now.b == per - 1 || done == run.to) {
                        if((uint32_t)col < rows)
#pragma unroll
                            for(int w = 0; w < 2; ++w)
#pragma unroll
                                for(int i = 0; i < 4; ++i)
                                    atomicAdd(&sums[now.item][w][col][4 * kg + i], acc[w][i]);
                        acc[0] = acc[1] = v4i{0, 0, 0, 0};
                    }
                    now.advance(per);
                }
            }
        }
        __syncthreads();

        // ---- SiLU(gate) * up: 16 threads a row of a tile ---------------------------
        for(uint32_t i = tid; i < (u1 - u0) * rows * kTile; i += kThreads) {
            const uint32_t j = i % kTile, r = i / kTile % rows, u = i / kTile / rows;
            const uint32_t c = (u0 - ai * tiles + u) * kTile + j;
            const float    rs = lds.scale[r];
            const float    g
                = ((float)sums[u][0][r][j] * rs) * a.sgu[(size_t)e * 2 * a.inter + c];
            const float v
                = ((float)sums[u][1][r][j] * rs) * a.sgu[(size_t)e * 2 * a.inter + a.inter + c];
            float f = silu_mul(g, v);
            if(a.s2) f *= a.s2[(size_t)e * a.inter + c];
            ws.act[(size_t)list[r] * a.inter + c] = f;
            f                                     = fabsf(f);
            f = fmaxf(f, dpp_mov<kDppQuadXor1>(f));
            f = fmaxf(f, dpp_mov<kDppQuadXor2>(f));
            f = fmaxf(f, dpp_mov<kDppRowHalfMirror>(f));
            f = fmaxf(f, dpp_mov<kDppRowMirror>(f));
            if(j == 0 && f > 0.f) atomicMax(&top[list[r]], __float_as_uint(f));
        }
        u0 = u1;
    }
    __syncthreads();
    for(uint32_t p = tid; p < pairs; p += kThreads)
        ws.top[(size_t)range * pairs + p] = __uint_as_float(top[p]);
}

// BLOCKS a CU.  Batches ahead: 3 where a block is alone on its CU, 2 where there are
// two; 7 and 3 of them made it slower (8 experts of 4096 x 14336, one token, 85 us against
// 80), as they have to where each batch waits for all of them.
template <bool F16, int BLOCKS>
__global__ void __launch_bounds__(kThreads, 2 * BLOCKS)
    gate_up_kernel(MoeDecodeArgs a, Ws ws, uint32_t group)
{
    extern __shared__ uint8_t dyn[];
    __shared__ GateUpLds      lds;
    gate_up<F16, BLOCKS == 1 ? 4 : 3>(a, ws, group, lds, dyn);
}

// ---------------------------------------------------------------------------
// Second kernel: the activations in 8 bits, once for all blocks of the third, 16 columns
// a thread of one pair's row a block row.  (Every block of the third kernel quantizing
// the rows for itself, into LDS: one token of 8 experts of 4096 x 14336 78 us the layer,
// 75 now; 16 tokens, whose rows did not fit, 308 and 256.)
// ---------------------------------------------------------------------------
constexpr int kRequantThreads = 256;

__global__ void __launch_bounds__(kRequantThreads)
    requant_kernel(MoeDecodeArgs a, Ws ws, uint32_t gu_blocks)
{
    __shared__ float tops[kRequantThreads / kWave];
    const uint32_t   tid = threadIdx.x, pairs = a.tokens * a.topk, p = blockIdx.y;
    const uint32_t   k = (blockIdx.x * kRequantThreads + tid) * 16;
    const float*     h = ws.act + (size_t)p * a.inter + k;
    v4f              f[4] = {};
#pragma unroll
    for(int c = 0; c < 4; ++c)
        if(k < a.inter) f[c] = *reinterpret_cast<const v4f*>(h + 4 * c);
    // (0 for a row of no expert, whose activations are whatever was there)
    static_assert(kGateUpBlocks <= 2 * kRequantThreads, "two maxima a thread");
    const uint32_t b = tid + kRequantThreads;
    const float    m0 = tid < gu_blocks ? ws.top[tid * pairs + p] : 0.f;
    const float    m1 = b < gu_blocks ? ws.top[b * pairs + p] : 0.f;
    float          m  = wave_max(fmaxf(m0, m1));
    if(tid % kWave == 0) tops[tid / kWave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    const float r = m / a.qmax, inv = r > 0.f ? 1.f / r : 0.f;
    v4i         w;
#pragma unroll
    for(int c = 0; c < 4; ++c)
        w[c] = (int)cvt_pack4_i8(quant_f(f[c][0], inv, a.qmax), quant_f(f[c][1], inv, a.qmax),
                                 quant_f(f[c][2], inv, a.qmax), quant_f(f[c][3], inv, a.qmax));
    if(k < a.inter) *reinterpret_cast<v4i*>(ws.q + (size_t)p * a.inter + k) = w;
    if(blockIdx.x == 0 && tid == 0) ws.scale[p] = r;
}

// ---------------------------------------------------------------------------
// Third kernel: a block owns 16 / FOLD output columns of all active experts.
// FOLD > 1 (at most 16 / FOLD tokens): the tile's 16 weight rows are the columns'
// FOLD parts along K, and its 16 columns the rows' parts likewise; the blocks on the
// tile's diagonal are the partial sums, the others are not used.  So a small hidden
// size still gives a block to every CU, with whole 16-byte loads.
// The quantized rows come as operands straight from L2, beside the weights: that is as
// many loads again, but no LDS, no barrier and nothing that every block does anew.
// ---------------------------------------------------------------------------
template <int FOLD, int RING, int kSteps>
__device__ __forceinline__ void down(const MoeDecodeArgs& a, const Ws& ws, uint8_t* dyn)
{
    constexpr uint32_t kCols = kTile / FOLD;
    const int      wave  = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int      lane  = threadIdx.x % kWave, col = lane % 16, kg = lane / 16;
    const uint32_t pairs = a.tokens * a.topk, tid = threadIdx.x;
    Lists          lists(dyn, pairs);
    int32_t*       sums = reinterpret_cast<int32_t*>(dyn + Lists::bytes(pairs)); // [pairs][kCols]
    const uint32_t j0   = blockIdx.x * kCols;

    const uint32_t n = (uint32_t)__builtin_amdgcn_readfirstlane(*ws.active);
    for(uint32_t i = tid; i < Lists::bytes(pairs) / 16; i += kThreads)
        reinterpret_cast<v4i*>(dyn)[i] = reinterpret_cast<const v4i*>(ws.lists)[i];
    for(uint32_t i = tid; i < pairs * kCols; i += kThreads) sums[i] = 0;
    __syncthreads();

    // ---- the stream of weights, all experts in one run a wave ------------------------
    const uint32_t part = ((a.inter + 63) / 64 + FOLD - 1) / FOLD; // steps of a part of K
    const uint32_t per  = (part + kSteps - 1) / kSteps;
    const Run      run(n * per, wave);
    const uint32_t mine = run.to - run.from;
    v4i            weights[RING][kSteps], rows[RING][kSteps];
    Cursor         ahead(run.from, per), now = ahead;
    const uint32_t row = col % kCols, fold = col / kCols; // of the weights, and of the tokens
    uint32_t       loaded = 0, item = ~0u, from = 0;
    const __amdgpu_buffer_rsrc_t rq = __builtin_amdgcn_make_buffer_rsrc(
        ws.q, 0, (int)(pairs * a.inter), kBufferFlags);
    auto load = [&](int slot) {
        const uint32_t               e = lists.expert_at(ahead.item);
        const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<int8_t*>(a.wd + ((size_t)e * a.hidden + j0) * a.inter), 0,
            (int)(kCols * a.inter), kBufferFlags);
        if(ahead.item != item) { // lanes past the expert's rows take its last one
            item = ahead.item;
            from = lists.pair[item * kRows + min(row, lists.rows(item) - 1)] * a.inter;
        }
#pragma unroll
        for(int i = 0; i < kSteps; ++i) {
            const uint32_t st = ahead.b * kSteps + i, k = (fold * part + st) * 64 + kg * 16;
            const bool     in = st < part && k < a.inter;
            weights[slot][i]  = load_weights(rw, in ? row * a.inter + k : kOob);
            rows[slot][i]     = load_weights(rq, in ? from + k : kOob);
        }
        ahead.advance(per);
        ++loaded;
    };
#pragma unroll
    for(int i = 0; i < RING - 1; ++i)
        if(loaded < mine) load(i);

    v4i acc = {};
    for(uint32_t done = 0; done < mine;) {
#pragma unroll
        for(int slot = 0; slot < RING; ++slot) {
            if(loaded < mine) load((slot + RING - 1) % RING);
            if(done < mine) {
#pragma unroll
                for(int i = 0; i < kSteps; ++i) acc = mfma(weights[slot][i], rows[slot][i], acc);
                ++done;
                const uint32_t ai = now.item;
                now.advance(per);
                if(now.item != ai || done == mine) {
                    if(row < lists.rows(ai) && (uint32_t)(4 * kg) / kCols == fold) {
                        int32_t* to = sums + lists.pair[ai * kRows + row] * kCols;
#pragma unroll
                        for(int i = 0; i < 4; ++i) atomicAdd(&to[(4 * kg + i) % kCols], acc[i]);
                    }
                    acc = v4i{0, 0, 0, 0};
                }
            }
        }
    }
    __syncthreads();

    // ---- the weighted sum over a token's slots -------------------------------------
    for(uint32_t i = tid; i < a.tokens * kCols; i += kThreads) {
        const uint32_t t = i / kCols, j = i % kCols;
        float          out = 0.f;
        for(uint32_t s = 0; s < a.topk; ++s) {
            const uint32_t p = t * a.topk + s;
            const int32_t  e = lists.ids[p];
            if(e < 0) continue;
            const float y
                = ((float)sums[p * kCols + j] * ws.scale[p]) * a.sd[(size_t)e * a.hidden + j0 + j];
            out = fmaf(ws.weight[p], y, out);
        }
        a.out[(size_t)t * a.ldo + j0 + j] = float_to_half_bits(out);
    }
}

// BLOCKS a CU, as in gate_up_kernel.  A batch is 4 steps, 4 KB a wave, or 2 where two
// blocks a CU leave no registers for 4 of weights and rows (16 tokens of 64 experts of
// 7168 x 2048, top 6, 394 us against 408; one block, 8 experts of 4096 x 14336: 4 steps
// 253 us, 2 steps 274).
template <int FOLD, int BLOCKS>
__global__ void __launch_bounds__(kThreads, 2 * BLOCKS) down_kernel(MoeDecodeArgs a, Ws ws)
{
    extern __shared__ uint8_t dyn[];
    down<FOLD, BLOCKS == 1 ? 4 : 3, BLOCKS == 1 ? 4 : 2>(a, ws, dyn);
}

template <class K>
void allow_lds(K kernel, uint32_t bytes)
{
    if(bytes + 32 * 1024 > 64 * 1024) // with the static part
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                  hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
}

template <int FOLD>
hipError_t launch_down(const MoeDecodeArgs& a, const Ws& ws, hipStream_t stream)
{
    const uint32_t pairs = a.tokens * a.topk, grid = a.hidden / (kTile / FOLD);
    const uint32_t lds    = Lists::bytes(pairs) + pairs * kTile * 4;
    const auto     kernel = grid <= kCus ? down_kernel<FOLD, 1> : down_kernel<FOLD, 2>;
    allow_lds(kernel, lds);
    kernel<<<grid, kThreads, lds, stream>>>(a, ws);
    return hipGetLastError();
}

} // namespace

size_t moe_ffn_decode_workspace_bytes(uint32_t tokens, uint32_t topk, uint32_t hidden,
                                      uint32_t inter)
{
    const size_t n = (size_t)tokens * topk;
    return up256(n * inter * 4) + up256(n * kGateUpBlocks * 4)
           + up256(Lists::bytes((uint32_t)n)) + 256 + 2 * up256(n * 4) + up256(n * inter);
}

hipError_t launch_moe_ffn_decode(const MoeDecodeArgs& a, bool f16, hipStream_t stream)
{
    const Ws       ws    = carve(a);
    const uint32_t pairs = a.tokens * a.topk;
    // 8 tiles' sums at a time, or 4 where two blocks then share a CU, or where 8 do not fit
    const uint32_t rest = Lists::bytes(pairs) + Lists::up16(pairs)
                          + a.tokens * row_bytes(a.hidden) + sizeof(GateUpLds);
    const uint32_t sum  = sizeof(TileSums);
    const bool     two  = rest + 4 * sum <= kLdsBytes / 2;
    const uint32_t group = rest + 8 * sum <= (two ? kLdsBytes / 2 : kLdsBytes) ? 8 : 4;
    const uint32_t lds   = rest - sizeof(GateUpLds) + group * sum;
    // as many blocks as are resident at once
    const uint32_t blocks = std::min(two ? kGateUpBlocks : kCus,
                                     std::min(pairs, a.experts) * (a.inter / kTile));
    const auto     gu     = f16 ? (two ? gate_up_kernel<true, 2> : gate_up_kernel<true, 1>)
                                : (two ? gate_up_kernel<false, 2> : gate_up_kernel<false, 1>);
    allow_lds(gu, lds);
    gu<<<blocks, kThreads, lds, stream>>>(a, ws, group);
    constexpr uint32_t kColumns = kRequantThreads * 16;
    const dim3         grid((a.inter + kColumns - 1) / kColumns, pairs);
    requant_kernel<<<grid, kRequantThreads, 0, stream>>>(a, ws, blocks);
    const hipError_t e = hipGetLastError();
    if(e != hipSuccess) return e;
    // a block for every CU, where the tokens leave room in the tile
    const uint32_t columns = a.hidden / kTile;
    if(columns < 128 && a.tokens <= 4) return launch_down<4>(a, ws, stream);
    if(columns < 256 && a.tokens <= 8) return launch_down<2>(a, ws, stream);
    return launch_down<1>(a, ws, stream);
}

} // namespace w8a8
