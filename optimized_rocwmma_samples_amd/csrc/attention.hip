// attention.hip -- causal attention of whole prompts for gfx950.
//
//   out[t, h] = sum_{j <= t} p[j] v[j],  p = softmax of scale * (q[t, h] . k[j])
//
// One pass over the keys with a running maximum m and sum l per query row.  A
// block owns 128 query rows of one head, 32 per wave, and walks the key tiles from the
// diagonal down to the sequence's first.
//   * Scores are computed transposed, S^T = K Q^T with v_mfma_f32_32x32x16_f16
//     (srcA = keys, srcB = queries): a lane then holds 16 of 32 keys' scores of
//     ONE query row (lane % 32), so maximum, exponential, sum and the rescaling
//     of the result are in-lane but for one exchange between the wave's halves,
//     and the probabilities, rounded to fp16, already are the srcB operand of
//     O^T += V^T P^T: the order in which that product takes the keys is free, so
//     a lane's registers are taken as they lie (key 8 (i / 4) + 4 (lane / 32) +
//     i % 4 in register i) and V^T is read to match.
//   * V^T comes out of a row-major tile in LDS with ds_read_b64_tr_b16: 16 lanes
//     read 4 keys x 16 channels and get 4 keys of one channel each.
//   * Key and value tiles go from global memory to LDS without registers, one tile
//     ahead, 16 bytes a lane; the 16-byte chunks of a row are stored XOR-swizzled
//     (chosen by the global address each lane fetches), so that both kinds of
//     reads spread over all banks.  Rows past the sequence's end read as zeros.
//   * The tile on the diagonal comes first and is the only one that masks.
// A tile of 32 keys of 128 channels is 512 cycles of products a wave and about as many of
// exponentials (a quarter of the rate), sums, maxima and roundings, which 3 waves a SIMD
// overlap in part.  8192 tokens, 32 query and 8 key heads of 128: 535 to 580 us by the
// card's clock, 1030 to 950 TFLOP/s, the matrix unit busy in 55 % of the cycles, vector
// instructions in 53 %, waves waiting for 23 % of their time; 16 heads of 64: 161 to 172 us.
// Bound, where blocks are few, by the chain of a block's own steps: key fragments come from LDS
// four ahead of their products, fragments of values each just before its own.  A block alone
// on its CU takes 1.2 us for 64 keys, whose products are half of that, which is what a prompt
// of 1024 tokens waits for.
#include "attention_tile.hpp"

namespace w8a8 {
namespace {

// Where a block works: one sequence's rows and a tile of kRows of them.
struct Span {
    uint32_t begin, len, tile;
    bool     live;
};

__device__ __forceinline__ uint32_t wave_sum(uint32_t v)
{
    int s = (int)v;
    s += dpp_mov_i32<kDppQuadXor1>(s);
    s += dpp_mov_i32<kDppQuadXor2>(s);
    s += dpp_mov_i32<kDppRowHalfMirror>(s);
    s += dpp_mov_i32<kDppRowMirror>(s);
    return (uint32_t)(__builtin_amdgcn_readlane(s, 0) + __builtin_amdgcn_readlane(s, 16)
                      + __builtin_amdgcn_readlane(s, 32) + __builtin_amdgcn_readlane(s, 48));
}

// Rows of a sequence: none where its starts do not ascend.
__device__ __forceinline__ void rows_of(const AttentionArgs& a, uint32_t i, int32_t& b, int32_t& e)
{
    b = e = 0;
    if(i < a.seqs) {
        b = min(max(a.starts[i], 0), (int32_t)a.tokens);
        e = max(min(max(a.starts[i + 1], 0), (int32_t)a.tokens), b);
    }
}

__device__ __forceinline__ uint32_t tiles_of(int32_t b, int32_t e)
{
    return (uint32_t)(e - b + kRows - 1) / kRows;
}

// Up to 64 sequences, one a lane: the tiles with the most keys of all sequences come
// first.  A sequence has a tile on each of its levels (a tile's place in it), so those
// above level x are sum(max(tiles - 1 - x, 0)), and the tile's level is found by halving.
// (Sequences one after the other: four of 2048 tokens, 32/8 heads of 128, 172 us, now
// 165; 8 x 512 tokens, 16 heads of 64, 14.9 and 14.1.)
__device__ __forceinline__ Span find_tile_of_few(const AttentionArgs& a, uint32_t tile, int lane)
{
    int32_t b, e;
    rows_of(a, lane, b, e);
    const uint32_t n = tiles_of(b, e);
    if(wave_sum(n) <= tile) return {0, 0, 0, false};
    uint32_t level = 0, above = (uint32_t)wave_max((float)n); // n is exact: below 2^24
    while(above - level > 1) {
        const uint32_t x = (level + above) / 2;
        if(wave_sum(n > x ? n - x : 0) > tile)
            level = x;
        else
            above = x;
    }
    // the level's tiles in the order of the sequences
    const uint32_t at   = tile - wave_sum(n > level ? n - level - 1 : 0);
    const uint64_t with = __ballot(n > level);
    const uint32_t rank = __builtin_popcountll(with & ((1ull << lane) - 1));
    const int      f    = __builtin_ctzll(__ballot(n > level && rank == at));
    const uint32_t bf = __builtin_amdgcn_readlane(b, f), ef = __builtin_amdgcn_readlane(e, f);
    return {bf, ef - bf, level, true};
}

// Any number of sequences: the tile-th tile of kRows query rows, 64 sequences a step,
// their tile counts summed along the lanes.  Inside a sequence the tiles with the most
// keys come first; the sequences keep their order, so a long one at the end starts last
// (64 tokens and a prompt of 4096, 16 heads of 64: 63 us, 60 with the prompt first).
__device__ __forceinline__ Span find_tile(const AttentionArgs& a, uint32_t tile, int lane)
{
    if(a.seqs <= kWave) return find_tile_of_few(a, tile, lane);
    uint32_t before = 0;
    for(uint32_t i0 = 0; i0 < a.seqs; i0 += kWave) {
        int32_t b, e;
        rows_of(a, i0 + lane, b, e);
        const uint32_t n = tiles_of(b, e);
        uint32_t       s = n;
#pragma unroll
        for(int d = 1; d < kWave; d <<= 1) {
            const uint32_t o = __shfl_up(s, d, kWave);
            if(lane >= d) s += o;
        }
        const uint64_t past = __ballot(before + s > tile);
        if(past != 0) {
            const int      f  = __builtin_ctzll(past);
            const uint32_t nf = __builtin_amdgcn_readlane(n, f);
            const uint32_t lo = before + __builtin_amdgcn_readlane(s, f) - nf;
            const uint32_t bf = __builtin_amdgcn_readlane(b, f);
            const uint32_t ef = __builtin_amdgcn_readlane(e, f);
            return {bf, ef - bf, nf - 1 - (tile - lo), tile >= lo && tile - lo < nf};
        }
        before += __builtin_amdgcn_readlane(s, kWave - 1);
    }
    return {0, 0, 0, false};
}

template <int D, int KEYS>
__device__ __forceinline__ void attention_rows(const AttentionArgs& a, uint8_t* lds)
{
    constexpr int kBlocks = D / 32; // 32-channel blocks of the result
    const int     lane    = threadIdx.x % kWave;

    // Blocks go round the 8 XCDs: where the heads divide evenly, an XCD gets
    // neighbouring heads, whose keys and values then stay in its L2.
    // Heads of 64: every other full round of one block a CU is turned around (inside each
    // XCD), so that tiles of many and of few keys share a CU and not like with like (key
    // tiles of 128, 2 blocks a CU: 8 x 512 tokens, 16 heads, 13.8 -> 13.0 us, 4096 tokens
    // 57 -> 55.5; key tiles of 64, 4 blocks: 8192 tokens 181 -> 170).
    // With heads of 128, 3 blocks a CU, it takes 2 % more.
    uint32_t block = blockIdx.x;
    if(D == 64 && block / kCus % 2 == 1 && (block / kCus + 1) * kCus <= gridDim.x)
        block ^= kCus - 8;
    uint32_t head = block % a.heads;
    if(a.heads % 8 == 0) head = head % 8 * (a.heads / 8) + head / 8;
    const Span span = find_tile(a, block / a.heads, lane);
    if(!span.live) return;
    const uint32_t kvh  = head / (a.heads / a.kv_heads);
    const uint32_t row0 = span.tile * kRows; // the block's first row in the sequence

    TileRows t;
    t.q     = a.q + (size_t)(span.begin + row0) * a.ldq + head * D;
    t.k     = a.k + (size_t)span.begin * a.ldk + kvh * D;
    t.v     = a.v + (size_t)span.begin * a.ldv + kvh * D;
    t.ldq   = a.ldq;
    t.ldk   = a.ldk;
    t.ldv   = a.ldv;
    t.rows  = min((uint32_t)kRows, span.len - row0);
    t.first = row0;
    t.keys  = span.len;
    t.from  = 0;
    t.to    = (row0 + t.rows + KEYS - 1) / KEYS; // tiles the block's rows see
    const float c = a.scale * 1.44269504088896341f;
    float       m = -INFINITY, l = 0.f, mc = 0.f;
    v16f        o[kBlocks] = {};
    attend<D, KEYS, false>(t, c, nullptr, lds, m, l, mc, o);
    const uint32_t row = threadIdx.x / kWave * 32 + lane % 32;
    write_rows(t.rows, row, l, o, a.out + (size_t)(span.begin + row0 + row) * a.ldo + head * D);
}

template <int D, int KEYS>
__global__ void __launch_bounds__(kThreads, (kBlocksOf<D, KEYS>)) attention_kernel(AttentionArgs a)
{
    __shared__ alignas(256) uint8_t lds[2 * 2 * KEYS * D * 2]; // two stages of keys, values
    attention_rows<D, KEYS>(a, lds);
}

} // namespace

hipError_t launch_attention(const AttentionArgs& a, hipStream_t stream)
{
    // no more tiles than full ones of all rows and one partial per sequence
    const uint32_t blocks = (a.tokens / kRows + a.seqs) * a.heads;
    // With few blocks a CU the time is a block's own, tile after tile, and the larger tiles
    // take less of it per key; with many the smaller ones' third wave fills the gaps.
    // us at tiles of 4096 / D and 8192 / D keys:
    //   heads of 128, one sequence: 2048 tokens, 8 heads 55.1, 45.5; 32 heads (544 blocks)
    //   61.1, 53.7; 4096 tokens, 32 heads (1056) 156, 161; 8192 tokens 616, 656
    //   several, any of which may be the long one: 1 to 2047 tokens, 32 heads (1184) 75.5,
    //   68.7; 8 x 512 (1280) 39.6, 39.7; 4 x 2048 (2176) 163, 168
    //   heads of 64: 4096 tokens, 16 heads (528) 59.9, 55.2; 8 x 512 (640) 13.2, 12.8; 4 x
    //   2048 (1088) 49.8, 55.3; 61 tokens, whose keys are one smaller tile, 4.7, 5.5
    // (The sequences' lengths are on the device: the mean stands for them, and a long
    // prompt beside many of a token takes the smaller tiles; 4096 and 63 of one: 61.)
    const uint32_t most = a.dim == 128 && a.seqs > 1 ? 5 * kCus : 3 * kCus;
    const bool     few  = blocks <= most && (a.dim == 128 || a.tokens / a.seqs > 128);
    const auto     kernel
        = a.dim == 64 ? (few ? attention_kernel<64, 128> : attention_kernel<64, 64>)
                      : (few ? attention_kernel<128, 64> : attention_kernel<128, 32>);
    kernel<<<blocks, kThreads, 0, stream>>>(a);
    return hipGetLastError();
}

} // namespace w8a8
