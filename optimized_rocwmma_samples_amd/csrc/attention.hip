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
// overlap in part.  8192 tokens, 32 query and 8 key heads of 128: 545 to 590 us by the
// card's clock, 1010 to 930 TFLOP/s, the matrix unit busy in 54 % of the cycles, vector
// instructions in 52 %, waves waiting for 31 % of their time; 16 heads of 64: 161 to 172 us.
// Bound, where blocks are few, by the chain of a block's own steps: the score product's key
// fragments come from LDS into one register quad (two for two chains), so that each product
// waits for its own read.  A block alone on its CU takes 1.2 us for 64 keys, whose products
// are half of that, which is what a prompt of 1024 tokens waits for (26 us).
#include "w8a8_device.hpp"
#include "w8a8_internal.hpp"

namespace w8a8 {
namespace {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float    v2f __attribute__((ext_vector_type(2)));
typedef float    v16f __attribute__((ext_vector_type(16)));
typedef __fp16   v4fp16 __attribute__((ext_vector_type(4)));

typedef __attribute__((address_space(3))) v4fp16 lds_v4h_t;
typedef __attribute__((address_space(3))) v8h    lds_v8h_t;

constexpr int kBufferFlags = 0x00020000; // raw buffer, 32-bit data format
constexpr int kRows        = 128;        // query rows a block
constexpr int kWaves       = kRows / 32;
constexpr int kThreads     = kWaves * kWave;
constexpr uint32_t kCus    = 256;

// Blocks a CU.  Keys a tile are 4096 / D, whose scores leave registers for 3 waves a SIMD
// and more, or twice as many, two independent chains a wave, for 2.
template <int D, int KEYS>
constexpr int kBlocksOf = D * KEYS == 4096 ? 3 : 2;

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

// The 16-byte chunk position of chunk c of row `tok` (an involution in c).
template <int D>
__device__ __forceinline__ uint32_t key_chunk(uint32_t tok, uint32_t c)
{
    return c ^ (D == 128 ? tok % 16 : tok / 2 % 8);
}

template <int D>
__device__ __forceinline__ uint32_t value_chunk(uint32_t tok, uint32_t c)
{
    return c ^ (D == 128 ? tok % 4 * 4 : tok / 2 % 2 * 4);
}

__device__ __forceinline__ v16f mfma(v8h a, v8h b, v16f c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// The value of the other half of the wave (lane ^ 32) and this one's.
__device__ __forceinline__ v2f both_halves(float v)
{
    const uint32_t u = __float_as_uint(v);
    const auto     r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return {__uint_as_float(r[0]), __uint_as_float(r[1])};
}

// max(a, b, c), NaN if one is: unlike fmaxf this takes no canonicalizing steps.  (Not in
// inline asm, which the compiler does not keep apart from the matrix operations before it.)
__device__ __forceinline__ float max3(float a, float b, float c)
{
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

__device__ __forceinline__ bool nonfinite(uint32_t h16) { return (h16 & 0x7C00u) == 0x7C00u; }

// The fp16 values of a fragment with infinities and NaN as 0.
__device__ __forceinline__ v8h finite_only(v8h v)
{
    v4i u = __builtin_bit_cast(v4i, v);
#pragma unroll
    for(int i = 0; i < 4; ++i) {
        const uint32_t w = (uint32_t)u[i];
        u[i] = (int)((nonfinite(w) ? 0u : w & 0xFFFFu)
                     | (nonfinite(w >> 16) ? 0u : w & 0xFFFF0000u));
    }
    return __builtin_bit_cast(v8h, u);
}

// From here on the wave's conversions to fp16 give +-65504 where a finite value passes the
// range (the mode register's FP16_OVFL; infinities and NaN stay what they are).  Matrix
// instructions lose NaN operands in this mode, so it begins behind those whose results `o`
// are; the converted values have to depend on the returned v.
template <int N>
__device__ __forceinline__ float finite_halves_from_here(float v, v16f (&o)[N])
{
#pragma unroll
    for(int i = 0; i < N; ++i) asm volatile("" : "+v"(o[i]));
    asm volatile("s_setreg_imm32_b32 hwreg(HW_REG_MODE, 23, 1), 1" : "+v"(v));
    return v;
}

// Twice 16 bytes a lane from a buffer into LDS, lane i to bytes `to` + 16 i and, from its
// second offset, 1024 further, with the caller's own waits: a load through the builtin makes
// the compiler wait for all of them ahead of every transposed read, whichever stage that
// reads.  The compiler does not see what asm reads, so the block itself keeps the five wait
// states between a vector instruction that writes a scalar register, such as the
// readfirstlane of a descriptor, and a memory instruction that reads it.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm" // m0 is reserved: set and used here alone
__device__ __forceinline__ void load_lds(v4i rsrc, uint32_t to, uint32_t offset0,
                                         uint32_t offset1)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %3, 0 offen lds\n\t"
                 "s_add_u32 m0, %0, 1024\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds"
                 :
                 : "s"(to), "v"(offset0), "v"(offset1), "s"(rsrc)
                 : "memory", "m0", "scc");
}
#pragma clang diagnostic pop

__device__ __forceinline__ v4i buffer(const void* base, uint32_t bytes)
{
    const uint64_t at = (uint64_t)base; // uniform, which the compiler does not always see
    return v4i{__builtin_amdgcn_readfirstlane((int)(uint32_t)at),
               __builtin_amdgcn_readfirstlane((int)((uint32_t)(at >> 32) & 0xFFFFu)),
               __builtin_amdgcn_readfirstlane((int)bytes), kBufferFlags};
}

template <int D, int kKeys>
__device__ __forceinline__ void attention_rows(const AttentionArgs& a, uint8_t* lds)
{
    constexpr int kSubs      = kKeys / 32;
    constexpr int kTileBytes = kKeys * D * 2;
    constexpr int kChunks    = D / 8;                  // 16-byte chunks per row
    constexpr int kRowsLoad  = kWave / kChunks;        // rows one wave-load fills
    constexpr int kLoads     = kKeys / kRowsLoad / kWaves; // wave-loads per wave and operand
    constexpr int kSteps     = D / 16;                 // MFMAs along the channels
    constexpr int kBlocks    = D / 32;                 // 32-channel blocks of the result
    static_assert(kLoads % 2 == 0, "wave-loads go in pairs");
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave, col = lane % 32, half = lane / 32;

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
    const uint32_t kvh   = head / (a.heads / a.kv_heads);
    const uint32_t row0  = span.tile * kRows;        // the block's first row in the sequence
    const uint32_t first = row0 + wave * 32;         // the wave's
    const uint32_t qi    = first + col;              // the lane's
    const uint32_t rows  = min((uint32_t)kRows, span.len - row0);

    // ---- tiles into LDS -------------------------------------------------------
    const uint32_t  ldkb = a.ldk * 2, ldvb = a.ldv * 2;
    const uint16_t* kbase = a.k + (size_t)span.begin * a.ldk + kvh * D;
    const uint16_t* vbase = a.v + (size_t)span.begin * a.ldv + kvh * D;
    uint32_t        ko[kLoads], vo[kLoads];
#pragma unroll
    for(int i = 0; i < kLoads; ++i) {
        const uint32_t tok = (wave * kLoads + i) * kRowsLoad + lane / kChunks;
        ko[i]              = tok * ldkb + key_chunk<D>(tok, lane % kChunks) * 16;
        vo[i]              = tok * ldvb + value_chunk<D>(tok, lane % kChunks) * 16;
    }
    const uint32_t lds0 = (uint32_t)(uintptr_t)lds;
    auto           issue = [&](int stage, uint32_t kt) {
        const uint32_t n = min((uint32_t)kKeys, span.len - kt * kKeys);
        const v4i      rk = buffer(kbase + (size_t)kt * kKeys * a.ldk, (n - 1) * ldkb + D * 2);
        const v4i      rv = buffer(vbase + (size_t)kt * kKeys * a.ldv, (n - 1) * ldvb + D * 2);
        const uint32_t to = lds0 + stage * 2 * kTileBytes + wave * kLoads * 1024;
#pragma unroll
        for(int i = 0; i < kLoads; i += 2) load_lds(rk, to + i * 1024, ko[i], ko[i + 1]);
#pragma unroll
        for(int i = 0; i < kLoads; i += 2)
            load_lds(rv, to + kTileBytes + i * 1024, vo[i], vo[i + 1]);
    };

    const uint32_t tiles = (row0 + rows + kKeys - 1) / kKeys; // tiles the block's rows see
    issue(0, tiles - 1);

    // ---- the wave's query rows: lane = row, 8 channels from 16 step + 8 half ----
    v8h qf[kSteps];
    {
        const __amdgpu_buffer_rsrc_t rq = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint16_t*>(a.q + (size_t)(span.begin + row0) * a.ldq + head * D), 0,
            (int)((rows - 1) * a.ldq * 2 + D * 2), kBufferFlags);
#pragma unroll
        for(int s = 0; s < kSteps; ++s)
            qf[s] = __builtin_bit_cast(
                v8h, __builtin_amdgcn_raw_buffer_load_b128(
                         rq, (wave * 32 + col) * a.ldq * 2 + s * 32 + half * 16, 0, 0));
    }

    // LDS places of the lane's reads, in stage 0: of a key's first step and a value's first
    // block.  Rows are D * 2 bytes and LDS starts on such a border, so the swizzle of a
    // later step or block is one XOR away; all else are fixed distances.
    const uint32_t kat = lds0 + col * D * 2 + key_chunk<D>(col, half) * 16;
    const uint32_t tok0 = 4 * half + lane % 16 / 4, ch0 = lane / 16 % 2 * 16 + lane % 4 * 4;
    const uint32_t vat
        = lds0 + kTileBytes + tok0 * D * 2 + value_chunk<D>(tok0, ch0 / 8) * 16 + ch0 % 8 * 2;

    const float c = a.scale * 1.44269504088896341f; // exponents in base 2
    float       m = -INFINITY, l = 0.f, mc = 0.f; // mc = m c, 0 while no score is finite
    v16f        o[kBlocks] = {};

    for(uint32_t step = 0; step < tiles; ++step) {
        const uint32_t kt    = tiles - 1 - step;
        const uint32_t stage = step % 2;
        wait_vmcnt<0>();   // this wave's part of the tile is there,
        wait_lgkmcnt0();   // and its reads of the tile before are done:
        __syncthreads();   // so are every wave's
        if(kt > 0) issue(stage ^ 1, kt - 1);
        if(kt * kKeys > first + 31) continue; // all of the tile is later than the wave's rows

        const uint32_t off  = stage * 2 * kTileBytes;
        const bool     diag = (kt + 1) * kKeys > first; // some of it is later than some rows
        v16f           s[kSubs] = {};
#pragma unroll
        for(int st = 0; st < kSteps; ++st)
#pragma unroll
            for(int sub = 0; sub < kSubs; ++sub)
                s[sub] = mfma(*(const lds_v8h_t*)(uintptr_t)(((kat + off) ^ (st * 32))
                                                             + sub * 32 * D * 2),
                              qf[st], s[sub]);
        if(diag) {
#pragma unroll
            for(int sub = 0; sub < kSubs; ++sub)
#pragma unroll
                for(int i = 0; i < 16; ++i) {
                    const uint32_t j = kt * kKeys + sub * 32 + 8 * (i / 4) + 4 * half + i % 4;
                    s[sub][i]        = j > qi ? -INFINITY : s[sub][i];
                }
        }
        float top = s[kSubs - 1][15];
#pragma unroll
        for(int i = 0; i < 16 * kSubs; i += 2)
            top = max3(top, s[i / 16][i % 16], s[(i + 1) / 16][(i + 1) % 16]);
        const v2f   tops = both_halves(top);
        const float mn   = fmaxf(m, fmaxf(tops[0], tops[1]));
        // m need not be the maximum itself: the result is rescaled only where some row's
        // probabilities would pass 2^8 (far inside fp16), which after the first tiles is
        // never, and not at every new maximum of one of 32 rows
        if(__ballot((mn - m) * c > 8.f) != 0) {
            const float next = mn == -INFINITY ? 0.f : mn * c;
            const float al   = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mc - next);
            m                = mn;
            mc               = next;
            l *= al;
#pragma unroll
            for(int b = 0; b < kBlocks; ++b) o[b] *= al;
        }

        // 4 keys of channel 32 b + col: keys 16 st + 8 part + 4 half ..
        auto values = [&](int b, int st) {
            v8h f;
#pragma unroll
            for(int part = 0; part < 2; ++part) {
                const auto r = __builtin_amdgcn_ds_read_tr16_b64_v4f16(
                    (lds_v4h_t*)(uintptr_t)(((vat + off) ^ (b * 64))
                                            + (16 * st + 8 * part) * D * 2));
#pragma unroll
                for(int i = 0; i < 4; ++i) f[part * 4 + i] = (_Float16)r[i];
            }
            return f;
        };
        v8h p[2 * kSubs];
#pragma unroll
        for(int st = 0; st < 2 * kSubs; ++st) {
#pragma unroll
            for(int i = 0; i < 8; i += 2) {
                const int   sub = st / 2, at = st % 2 * 8 + i;
                const float p0  = __builtin_amdgcn_exp2f(fmaf(s[sub][at], c, -mc));
                const float p1  = __builtin_amdgcn_exp2f(fmaf(s[sub][at + 1], c, -mc));
                l += p0;
                l += p1;
                const v2h h  = __builtin_convertvector((v2f{p0, p1}), v2h);
                p[st][i]     = h[0];
                p[st][i + 1] = h[1];
            }
#pragma unroll
            for(int b = 0; b < kBlocks; ++b) o[b] = mfma(values(b, st), p[st], o[b]);
        }

        if(diag) {
            // A masked probability is 0, but 0 times an infinity or NaN is not: where
            // the first product of the wave's rows (the diagonal comes first) is not
            // finite, take it again without such values and add each of them to
            // exactly the rows that see it.
            float z = 0.f;
#pragma unroll
            for(int b = 0; b < kBlocks; ++b)
#pragma unroll
                for(int i = 0; i < 16; ++i) z = fmaf(o[b][i], 0.f, z);
            if(__ballot(z != 0.f) != 0) {
#pragma unroll
                for(int b = 0; b < kBlocks; ++b) {
                    o[b] = v16f{};
#pragma unroll
                    for(int st = 0; st < 2 * kSubs; ++st)
                        o[b] = mfma(finite_only(values(b, st)), p[st], o[b]);
                }
                for(uint32_t tok = 0; tok < kKeys; ++tok) {
                    if(kt * kKeys + tok > qi) break;
#pragma unroll
                    for(int b = 0; b < kBlocks; ++b)
#pragma unroll
                        for(int i = 0; i < 16; ++i) {
                            const uint32_t ch = 32 * b + 8 * (i / 4) + 4 * half + i % 4;
                            const uint32_t v  = *(const __attribute__((address_space(3)))
                                                     uint16_t*)(uintptr_t)(
                                lds0 + off + kTileBytes + tok * D * 2
                                + value_chunk<D>(tok, ch / 8) * 16 + ch % 8 * 2);
                            if(nonfinite(v)) o[b][i] += half_bits_to_float(v);
                        }
                }
            }
        }
    }

    const v2f   ls  = both_halves(l);
    // The rounded probabilities may add up to a little more than l (2^-11 of it at the most),
    // which must not carry a mean of values of 65504 past fp16.
    const float inv = finite_halves_from_here(1.f / (ls[0] + ls[1]), o);
    if(qi >= span.len) return;
    uint16_t* out = a.out + (size_t)(span.begin + qi) * a.ldo + head * D;
#pragma unroll
    for(int b = 0; b < kBlocks; ++b)
#pragma unroll
        for(int i = 0; i < 16; i += 4) {
            v2i w;
            w[0] = (int)float2_to_half2_bits_2step(o[b][i] * inv, o[b][i + 1] * inv);
            w[1] = (int)float2_to_half2_bits_2step(o[b][i + 2] * inv, o[b][i + 3] * inv);
            *reinterpret_cast<v2i*>(out + 32 * b + 8 * (i / 4) + 4 * half) = w;
        }
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
