// kv4_chunks.hip -- attention of several new tokens per sequence over the paged 4-bit
// cache, for gfx950.
//
//   out[t, h] = sum_j p[j] v[j],  p = softmax of scale * (q[t, h] . k[j]) over the tokens j of
//   t's sequence up to t itself; the rows of q are the sequence's last tokens.
//
// Sequences of few rows are computed here, those of many in kv4_unpacked.hip (kFewRows in
// kv4_chunks.hpp).  The rows of a unit of work are (token, query head) pairs of one key head:
// row r is token r / per, head r % per, per query heads sharing the key head.  A unit has 32
// of them, or 64 where the sequence has more than 32 (24 x 5 tokens of 64/8 heads: 78 us in
// units of 32, 63 in units of 64, whose codes are unpacked once for both).  Units are walked
// in steps of 128 keys, 32 a wave.  The steps of the units of 64 rows lie in one line, those of
// 32 in another; each line is cut into up to 512 equal runs, a block each, two of which a CU
// holds, and the blocks of the first line start first.  What a cut leaves of a unit is written as
// partials (sum of p v, maximum and sum of p of each row) and joined by a second launch.
//   * S^T = K Q^T with v_mfma_f32_32x32x16_f16: srcA rows are keys, and a lane's operand is 8
//     channels of one key, which is a dword of its codes: unpacked, scaled and used where
//     it was loaded.  The queries lie in LDS in the order of the other operand.
//   * The scores of one query row lie in a lane (and lane ^ 32), so softmax stays there, and
//     the probabilities are the srcB operand of O^T += V^T P^T as they are.
//   * V^T's rows are channels: a wave unpacks its 32 rows of values into a tile of its own in
//     LDS and reads it transposed with ds_read_b64_tr_b16.  Nothing waits for other waves
//     until the unit ends.
// A code n becomes 512 + n / 2 by two bit operations a pair, (n - 8) / 2 and then offset / 2 +
// scale * (n - 8) / 2, rounded once: half of what kv4_load gives, since a group that reaches the
// ends of fp16 may pass them by half a step (the halves go into the scale of the scores and of
// the result).  Half of a subnormal offset is rounded as well, so that small values are off by
// up to 2^-23.  Three roundings of 2^-11 are left, of keys, values and probabilities, as in
// attention over fp16 keys and values.  Relative to the results' norm, 5 tokens verified and one
// decoded beside a prompt: keys 4.9e-4 and 3.0e-4, values 1.9e-4, probabilities 1.0e-4 and
// 0.7e-4, the results' own rounding 2.1e-4 and 2.0e-4; all of them 5.8e-4 and 4.0e-4.  That one
// token alone, by attention_kv4, is 2.0e-4 off: its codes enter as 1 + n / 16, exactly, with
// scales applied around the products, which here would take a product per group and query row
// and cost long chunks a quarter of their time; so a token that is decoded beside chunks is
// computed as they are.
//
// MI355X, 64 query and 8 key heads of 128, groups of 32: the last 5 tokens of 24 sequences of
// 978 to 7719 (137 MB of codes and scales) take 60 us of this kernel, 2.3 TB/s, and 9 of the join.
// Vector instructions fill 43 % of the SIMDs' cycles from the launch's start to its end, about
// half of them unpacking, matrix instructions 18 %; the rest is what two waves a SIMD wait for
// LDS, loads and each other's products, and the blocks' starts, unit ends and unequal ends.  One
// token of 131072 of 32/8 heads: 49 + 5 us.  Of equal runs of 13 steps those of the first 256
// blocks end after 44 us and the others, whose waves a SIMD serves second, after 54; a unit's end
// costs 5.  Not faster: codes staged through LDS by DMA (62, 57), keys unpacked ahead of values
// (72), three blocks a CU (spills), queries and values read one product ahead, longer runs for
// the first blocks, priorities that take turns.
#include "kv4_chunks.hpp"

#include <algorithm>

namespace w8a8 {
namespace {

typedef __attribute__((address_space(3))) v4i    lds_v4i_t;
typedef __attribute__((address_space(3))) v4f    lds_v4f_t;

constexpr int      kWaves   = 4;
constexpr int      kThreads = kWaves * kWave;
constexpr int      kKeys    = 32;              // a wave's a step
constexpr int      kStep    = kWaves * kKeys;  // keys of a step
constexpr uint32_t kBlocks  = 512;             // runs of a line at the most: two blocks a CU

__host__ __device__ inline uint32_t steps_of(uint32_t len)
{
    return len == 0 ? 1u : (len + kStep - 1) / kStep; // a sequence of no tokens is written too
}

__device__ __forceinline__ bool finite_pair(uint32_t w)
{
    return (w & 0x7C00u) != 0x7C00u && (w & 0x7C000000u) != 0x7C000000u;
}

// The 8 codes of a dword as fp16 values (offset + scale * (n - 8)) / 2, in the order 0 4 1 5 2 6
// 3 7; `pair` is (scale, offset / 2).
struct Unpack {
    uint32_t mask, big;
    __device__ Unpack()
    {
        asm volatile("v_mov_b32 %0, 0x000f000f" : "=v"(mask));
        asm volatile("v_mov_b32 %0, 0x60006000" : "=v"(big)); // 512, whose last bit is 1/2
    }
    __device__ v8h operator()(uint32_t w, v2h pair) const
    {
        const v2h middle = {(_Float16)516.f, (_Float16)516.f};
        const v2h s = {pair[0], pair[0]}, o = {pair[1], pair[1]};
        v8h       f;
#pragma unroll
        for(int i = 0; i < 4; ++i) {
            const v2h n = __builtin_bit_cast(v2h, ((w >> (4 * i)) & mask) | big) - middle;
            const v2h v = __builtin_elementwise_fma(n, s, o);
            f[2 * i]     = v[0];
            f[2 * i + 1] = v[1];
        }
        return f;
    }
};

// The scale as it is and half of the offset, x + 0 x and x - x / 2: infinities become NaN by it.
// (Half a scale that is subnormal in fp16 would be off by up to half a step, times 8.  The
// factors 0 and -1/2 are one inline constant; -0 or 1, 1/2 take a register, which spills.)
__device__ __forceinline__ v2h scale_and_half(int32_t pair)
{
    const v2h x = __builtin_bit_cast(v2h, pair);
    return __builtin_elementwise_fma(x, v2h{(_Float16)0.f, (_Float16)-0.5f}, x);
}

// The 16-byte chunk position of chunk c of a row of a wave's tile of values: spreads both the
// writes (lanes = rows) and the transposed reads (4 rows x 16 channels) over the banks.
template <int D>
__device__ __forceinline__ uint32_t value_chunk(uint32_t tok, uint32_t c)
{
    return c ^ (D == 128 ? tok % 4 * 4 : tok / 2 % 2 * 4) ^ (tok / 4 % 2);
}

// A step's keys and values on their way.
template <int D, int G>
struct Raw {
    static constexpr int kKeyWords   = D / 32;                         // of each of two places
    static constexpr int kValueWords = D / 16;                         // half a row
    static constexpr int kValuePairs = D / 2 / G == 0 ? 1 : D / 2 / G; // groups of half a row
    int32_t k[2][kKeyWords], v[kValueWords], ks[D / G], vs[kValuePairs];
    bool    ok; // the lane's key has a page
};

struct Place {
    uint32_t seq, unit, step, steps, tiles; // tiles: of the sequence's rows
    Chunk    c;
};

// A block's run: which steps of the line it takes, and where the first of them lies.
struct Line {
    uint32_t q, r;      // runs have q steps, the first r of them one more
    uint32_t left, end; // its steps, and the place on the line behind the last (of equal runs)
    uint32_t seq, at;   // the first one's sequence, and place in it
};

// What the launch's blocks are given, and the sequences' ways.
struct Ways {
    const uint8_t* others; // [seqs] 1: unpacked first; or null
    uint32_t       per, most;
    bool           more; // there are blocks for units of two tiles

    // 32-row tiles a unit; 0: not this kernel's
    __device__ uint32_t kind(const Chunk& x, uint32_t i) const
    {
        if(x.fresh == 0 || (others != nullptr && others[i] != 0)) return 0;
        return more && x.fresh * per > 32 ? 2 : 1;
    }
};

__device__ __forceinline__ uint32_t unit_tiles(const Chunk& x, uint32_t per, uint32_t kind)
{
    return (x.fresh * per + 32 * kind - 1) / (32 * kind);
}

// Run `run` of `runs` on the line of the sequences whose units are T tiles of 32 rows: equal
// runs, or one unit each.
template <int T>
__device__ __forceinline__ Line find_line(const ChunkArgs& a, const Ways& w, uint32_t kv_heads,
                                          uint32_t run, uint32_t runs)
{
    const uint32_t lane = threadIdx.x % kWave;
    uint32_t       n, units, steps, s;
    const auto     scan = [&](uint32_t i0) { // 64 sequences' steps
        const uint32_t i = i0 + lane;
        units = steps = 0;
        if(i < a.seqs) {
            const Chunk x = chunk_of(a, i, w.most);
            if(w.kind(x, i) == T) {
                units = unit_tiles(x, w.per, T) * kv_heads;
                steps = steps_of(x.len);
            }
        }
        n = units * steps;
        s = lanes_sum(n);
        return (uint32_t)__builtin_amdgcn_readlane((int)s, kWave - 1);
    };
    float    total = 0.f; // starts that do not ascend may count rows so often that sums wrap
    uint32_t all = 0, most_steps = 0, all_units = 0;
    for(uint32_t i = 0; i < a.seqs; i += kWave) {
        all += scan(i);
        total += wave_sum((float)n);
        most_steps = max(most_steps, (uint32_t)-wave_min_i32(-(int32_t)steps));
        all_units += __builtin_amdgcn_readlane((int)lanes_sum(units), kWave - 1);
    }
    if(total > 2147483648.f) all = 0;
    // One unit each where no unit has many steps more than an equal run: what is cut costs its
    // run's end and the join, some 5 to 10 us with many units, less with few; a step 2 to 3.
    // us cut and whole: 24 sequences of 256 tokens, 4 new ones each of 64/8 heads (192 units of
    // 2 steps) 17.9, 12.4, of 1024 (8 steps for 3) 27.1, 22.2; 4 of 768, 1 new of 32/8 (32 units
    // of 6 steps for 1) 14.5, 16.6.
    const bool whole
        = all_units <= runs && most_steps <= (all + runs - 1) / runs + min(5u, 1 + all_units / 32);
    Line l{};
    if(whole) {
        l.q    = 1;
        l.left = run < all_units && all != 0 ? 1 : 0;
    } else {
        l.q    = all / runs;
        l.r    = all % runs;
        l.left = l.q + (run < l.r ? 1 : 0);
    }
    uint32_t at = run * l.q + min(run, l.r);
    l.end       = at + l.left;
    if(l.left == 0) return l;
    for(uint32_t i = 0; i < a.seqs; i += kWave) {
        if(a.seqs > kWave) scan(i); // (of up to 64 sequences it is still there)
        if(whole) s = lanes_sum(units);
        const uint32_t sum = (uint32_t)__builtin_amdgcn_readlane((int)s, kWave - 1);
        if(at < sum) {
            const int f = __builtin_ctzll(__ballot(s > at));
            l.at = at - ((uint32_t)__builtin_amdgcn_readlane((int)s, f)
                         - (uint32_t)__builtin_amdgcn_readlane((int)(whole ? units : n), f));
            l.seq = i + f;
            if(whole) {
                l.left = __builtin_amdgcn_readlane((int)steps, f);
                l.at *= l.left;
            }
            break;
        }
        at -= sum;
    }
    return l;
}

template <int D, int G, int T>
__device__ __forceinline__ void chunks_run(const CacheView& c, const ChunkArgs& a, const Runs& runs,
                                           const Ways& ways, uint32_t run, uint32_t pages,
                                           uint8_t* lds, float* lds_ml)
{
    using R = Raw<D, G>;
    constexpr int  kSteps = D / 16, kBlk = D / 32; // products along the channels; result blocks
    constexpr int  kTile = kKeys * D * 2;          // bytes of a wave's values
    constexpr uint32_t kRows = 32 * T;             // rows of a unit
    const int      wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int      lane = threadIdx.x % kWave, col = lane % 32, half = lane / 32;
    const uint32_t per = ways.per;
    const uint32_t lds0 = (uint32_t)(uintptr_t)lds, tile = lds0 + wave * kTile;
    const uint32_t qat = lds0 + kWaves * kTile + lane * 16;

    const Line line = find_line<T>(a, ways, c.kv_heads, run, runs.count);
    uint32_t   tasks = 0; // that the join has with what this run cuts
    if(line.left == 0) {
        if(runs.cut && threadIdx.x == 0) runs.tasks[run] = 0;
        return;
    }
    uint32_t   left  = line.left;
    const auto enter = [&](Place& p) { // the sequence p.seq
        p.c     = chunk_of(a, p.seq, ways.most);
        p.steps = steps_of(p.c.len);
        p.tiles = ways.kind(p.c, p.seq) == T ? unit_tiles(p.c, per, T) : 0;
    };
    Place here{};
    here.seq = line.seq;
    enter(here);
    here.unit = line.at / here.steps;
    here.step = line.at % here.steps;
    auto advance = [&](Place& p) { // to the next step, whichever unit's; not past the run
        if(++p.step != p.steps) return;
        p.step = 0;
        if(++p.unit != p.tiles * c.kv_heads) return;
        p.unit = 0;
        do {
            ++p.seq;
            enter(p);
        } while(p.tiles == 0);
    };

    // ---- steps on their way ------------------------------------------------------------
    auto page_at = [&](const Place& p) { // of the lane's key, as it stands in the table
        const uint32_t t    = p.step * kStep + wave * kKeys + col;
        int32_t        page = -1;
        if(t < p.c.len) page = a.table[(size_t)p.seq * a.table_ld + (t >> c.page_shift)];
        return page;
    };
    auto fetch = [&](R& x, const Place& p, int32_t page) {
        x.ok             = (uint32_t)page < pages; // else page 0's rows are read, and masked
        const size_t row = cache_row(c, x.ok ? page : 0, p.unit / p.tiles,
                                     (p.step * kStep + wave * kKeys + col) & (c.page_size - 1));
        const uint8_t* k = c.codes[0] + row * (D / 2) + half * (D / 8);
        load_dwords<R::kKeyWords>(x.k[0], k);
        load_dwords<R::kKeyWords>(x.k[1], k + D / 4);
        load_dwords<D / G>(x.ks, c.scales[0] + row * (D / G));
        const uint8_t* v = c.codes[1] + row * (D / 2) + half * (D / 4);
#pragma unroll
        for(int i = 0; i < R::kValueWords; i += 4) load_dwords<4>(x.v + i, v + 4 * i);
        load_dwords<R::kValuePairs>(x.vs, c.scales[1] + row * (D / G) + half * (D / 2) / G);
    };

    // ---- the queries, in LDS as the products take them: [32 rows][product][lane] ---------
    uint32_t   sees[T] = {}, least = 0; // keys the lane's rows see, and the unit's first row
    v8h        qv[T][kSteps / kWaves];  // this wave's share of them on their way
    const auto fetch_queries = [&](const Place& p) {
        const uint32_t row0 = p.unit % p.tiles * kRows, rows = p.c.fresh * per;
        auto           seen = [&](uint32_t row) {
            return (uint32_t)max((int32_t)(p.c.len + row / per + 1 - p.c.fresh), 0);
        };
        least = seen(row0);
#pragma unroll
        for(int t = 0; t < T; ++t) {
            const uint32_t row = min(row0 + 32 * t + col, rows - 1);
            sees[t]            = seen(row);
            const uint16_t* from = a.q + (size_t)(p.c.begin + row / per) * a.ldq
                                   + (size_t)(p.unit / p.tiles * per + row % per) * D + 8 * half;
#pragma unroll
            for(int i = 0; i < kSteps / kWaves; ++i)
                qv[t][i] = *reinterpret_cast<const v8h*>(from + 16 * (wave + i * kWaves));
        }
    };
    const auto keep_queries = [&] {
        constexpr int kOrder[8] = {0, 4, 1, 5, 2, 6, 3, 7};
#pragma unroll
        for(int t = 0; t < T; ++t)
#pragma unroll
            for(int i = 0; i < kSteps / kWaves; ++i) {
                const v8h q = infinite_to_nan(qv[t][i]);
                v8h       u;
#pragma unroll
                for(int e = 0; e < 8; ++e) u[e] = q[kOrder[e]];
                *(lds_v4i_t*)(uintptr_t)(qat + (t * kSteps + wave + i * kWaves) * kWave * 16)
                    = __builtin_bit_cast(v4i, u);
            }
        __syncthreads();
    };

    const Unpack unpack;
    const float  c2 = a.scale * (2.f * 1.44269504088896341f); // base 2, of halved keys
    const uint32_t tok0 = 4 * half + lane % 16 / 4, ch0 = lane / 16 % 2 * 16 + lane % 4 * 4;
    const uint32_t vat  = tile + tok0 * D * 2 + value_chunk<D>(tok0, ch0 / 8) * 16 + ch0 % 8 * 2;

    // of each 32 rows: maximum, mc = m c2 (0 while no score is finite), sum, result
    float m[T], l[T], mc[T];
    v16f  o[T][kBlk];
    auto  begin_unit = [&] {
#pragma unroll
        for(int t = 0; t < T; ++t) {
            m[t]  = -INFINITY;
            mc[t] = 0.f;
            l[t]  = 0.f;
#pragma unroll
            for(int b = 0; b < kBlk; ++b) o[t][b] = v16f{};
        }
    };
    begin_unit();
    bool from_start = here.step == 0; // of the unit

    R     x;
    Place next = here, after{};
    {
        const int32_t page = page_at(here);
        fetch_queries(here);
        fetch(x, here, page);
    }
    int32_t page_next = -1, page_after = -1;
    if(left > 1) {
        advance(next);
        page_next = page_at(next);
    }
    keep_queries();

    // The waves' results of 32 rows joined and written, at the unit's end or the run's: a half
    // of them at a time is left in LDS, and each wave adds up a quarter of that.
    auto finish = [&](const int t, bool ends) {
        constexpr int kHalf = kBlk * 8, kMine = kBlk * 2; // registers
        const v2f     ls = both_halves(l[t]);
        const uint32_t row0 = here.unit % here.tiles * kRows + 32 * t, rows = here.c.fresh * per;
        const uint32_t row = row0 + col, head0 = here.unit / here.tiles * per;
        const size_t   slot = (size_t)(2 * run + (from_start ? 1 : 0)) * kRows + 32 * t + col;
        const bool     done = ends && from_start;
#pragma unroll
        for(int h = 0; h < 2; ++h) {
            __syncthreads(); // all waves are done with what lies there
            if(h == 0 && half == 0) {
                lds_ml[(wave * 32 + col) * 2]     = m[t];
                lds_ml[(wave * 32 + col) * 2 + 1] = ls[0] + ls[1];
            }
#pragma unroll
            for(int i = 0; i < kHalf; i += 4) {
                const int at = h * kHalf + i;
                *(lds_v4f_t*)(uintptr_t)(lds0 + (wave * kHalf + i) * kWave * 4 + lane * 16)
                    = v4f{o[t][at / 16][at % 16], o[t][at / 16][at % 16 + 1],
                          o[t][at / 16][at % 16 + 2], o[t][at / 16][at % 16 + 3]};
            }
            __syncthreads();
            float common = -INFINITY, sum = 0.f;
#pragma unroll
            for(int w = 0; w < kWaves; ++w) common = fmaxf(common, lds_ml[(w * 32 + col) * 2]);
            float r[kMine];
#pragma unroll
            for(int w = 0; w < kWaves; ++w) {
                const float mw = lds_ml[(w * 32 + col) * 2];
                const float f
                    = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mw - common) * c2);
                sum = fmaf(f, lds_ml[(w * 32 + col) * 2 + 1], sum);
#pragma unroll
                for(int i = 0; i < kMine; i += 4) {
                    const v4f u = *(lds_v4f_t*)(uintptr_t)(lds0 + w * (kHalf * kWave * 4)
                                                           + (wave * kMine + i) * kWave * 4
                                                           + lane * 16);
#pragma unroll
                    for(int e = 0; e < 4; ++e)
                        r[i + e] = w == 0 ? u[e] * f : fmaf(u[e], f, r[i + e]);
                }
            }
            const uint32_t ch0 = 2 * (h * kHalf + wave * kMine) + 4 * half;
            if(done) {
                const float inv = sum != 0.f ? 2.f / sum : 0.f;
                uint16_t*   out = a.out + (size_t)(here.c.begin + row / per) * a.ldo
                                + (size_t)(head0 + row % per) * D + ch0;
#pragma unroll
                for(int i = 0; i < kMine; i += 4) {
                    // this half has channels 0 1, 4 5 (2 3, 6 7) of a chunk of 8
                    const auto w = __builtin_amdgcn_permlane32_swap(
                        finite_halves(r[i] * inv, r[i + 2] * inv),
                        finite_halves(r[i + 1] * inv, r[i + 3] * inv), false, false);
                    if(row < rows)
                        *reinterpret_cast<v2i*>(out + 2 * i) = v2i{(int)w[0], (int)w[1]};
                }
            } else if(row < rows) {
#pragma unroll
                for(int i = 0; i < kMine; i += 4)
                    *reinterpret_cast<v4f*>(runs.o + slot * D + ch0 + 2 * i)
                        = v4f{r[i], r[i + 1], r[i + 2], r[i + 3]};
                if(h == 0 && half == 0 && wave == 0)
                    *reinterpret_cast<v2f*>(runs.ml + slot * 2) = v2f{common * c2, sum};
            }
        }
        if(t == 0 && !ends && from_start && threadIdx.x == 0) { // goes on behind the run
            const uint32_t last = line.end - 1 + (here.steps - 1 - here.step); // its last step
            const uint32_t q = line.q, r1 = line.r;
            const uint32_t to
                = last < r1 * (q + 1) ? last / (q + 1) : r1 + (last - r1 * (q + 1)) / q;
            runs.cut[run] = {to + 1, here.c.begin, row0, rows, head0, {}};
            tasks         = join_tasks<D>(to + 1 - run, min(kRows, rows - row0));
        }
    };

    for(; left > 0; --left) {
        const uint32_t key0 = here.step * kStep + wave * kKeys;
        const uint32_t live = (uint32_t)__ballot(x.ok); // keys that are there
        const bool     full = live == ~0u && key0 + kKeys <= least;

        // ---- values into LDS; NaN ones of keys that only some rows see are kept out -----
        uint64_t bad[R::kValuePairs] = {};
        v2h      vs[R::kValuePairs];
#pragma unroll
        for(int g = 0; g < R::kValuePairs; ++g) {
            if(!x.ok) x.vs[g] = 0;
            if(!full) {
                const bool nan = !finite_pair((uint32_t)x.vs[g]) && key0 + col >= least;
                bad[g]         = __ballot(nan);
                if(nan) x.vs[g] = 0;
            }
            vs[g] = scale_and_half(x.vs[g]);
        }
#pragma unroll
        for(int i = 0; i < R::kValueWords; ++i) {
            const v8h v = unpack((uint32_t)x.v[i], vs[i * 8 / G]);
            *(lds_v4i_t*)(uintptr_t)(tile + col * D * 2
                                     + value_chunk<D>(col, half * (D / 16) + i) * 16)
                = __builtin_bit_cast(v4i, v);
        }
        // ---- scores -----------------------------------------------------------------------
        v16f sc[T] = {};
#pragma unroll
        for(int st = 0; st < kSteps; ++st) {
            const v8h k = unpack((uint32_t)x.k[st % 2][st / 2], scale_and_half(x.ks[st / 2 * 32 / G]));
#pragma unroll
            for(int t = 0; t < T; ++t)
                sc[t] = mfma(k,
                             __builtin_bit_cast(v8h, *(lds_v4i_t*)(uintptr_t)(
                                                         qat + (t * kSteps + st) * kWave * 16)),
                             sc[t]);
        }
        // The next step's loads, over the rest of this one; before them the page numbers of the
        // step after it, which would else be waited for together with those loads (1 to 2 %).
        if(left > 1) {
            if(left > 2) {
                after = next;
                advance(after);
                page_after = page_at(after);
            }
            fetch(x, next, page_next);
        }
        if(!full)
#pragma unroll
            for(int i = 0; i < 16; ++i) {
                const uint32_t j = 8 * (i / 4) + 4 * half + i % 4;
#pragma unroll
                for(int t = 0; t < T; ++t)
                    if(key0 + j >= sees[t] || !((live >> j) & 1u)) sc[t][i] = -INFINITY;
            }
#pragma unroll
        for(int t = 0; t < T; ++t) {
            float top = sc[t][15];
#pragma unroll
            for(int i = 0; i < 16; i += 2) top = max3(top, sc[t][i], sc[t][i + 1]);
            const v2f   tops = both_halves(top);
            const float mn   = fmaxf(m[t], fmaxf(tops[0], tops[1]));
            // m need not be the maximum itself: rescaled only where probabilities would pass 2^8
            if(__ballot((mn - m[t]) * c2 > 8.f) != 0) {
                const float to = mn == -INFINITY ? 0.f : mn * c2;
                const float al = m[t] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mc[t] - to);
                m[t]           = mn;
                mc[t]          = to;
                l[t] *= al;
#pragma unroll
                for(int b = 0; b < kBlk; ++b) o[t][b] *= al;
            }
        }
        // ---- O^T += V^T P^T ----------------------------------------------------------------
#pragma unroll
        for(int st = 0; st < 2; ++st) {
            v8h p[T];
#pragma unroll
            for(int t = 0; t < T; ++t)
#pragma unroll
                for(int i = 0; i < 8; i += 2) {
                    const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[t][st * 8 + i], c2, -mc[t]));
                    const float p1
                        = __builtin_amdgcn_exp2f(fmaf(sc[t][st * 8 + i + 1], c2, -mc[t]));
                    l[t] += p0;
                    l[t] += p1;
                    const v2h h = __builtin_convertvector((v2f{p0, p1}), v2h);
                    p[t][i]     = h[0];
                    p[t][i + 1] = h[1];
                }
#pragma unroll
            for(int b = 0; b < kBlk; ++b) {
                v8h f; // 4 keys of channel 32 b + col (in the codes' order), and 4 more
#pragma unroll
                for(int part = 0; part < 2; ++part) {
                    const auto t = __builtin_amdgcn_ds_read_tr16_b64_v4f16(
                        (lds_v4h_t*)(uintptr_t)((vat ^ (b * 64)) + (16 * st + 8 * part) * D * 2));
#pragma unroll
                    for(int i = 0; i < 4; ++i) f[part * 4 + i] = (_Float16)t[i];
                }
#pragma unroll
                for(int t = 0; t < T; ++t) o[t][b] = mfma(f, p[t], o[t][b]);
            }
        }
        if(!full) { // NaN values, to exactly the rows that see them
#pragma unroll
            for(int g = 0; g < R::kValuePairs; ++g)
                for(uint64_t left_bad = bad[g]; left_bad != 0; left_bad &= left_bad - 1) {
                    const int f = __builtin_ctzll(left_bad), grp = f / 32 * (D / 2) / G + g;
#pragma unroll
                    for(int t = 0; t < T; ++t)
                        if(key0 + f % 32 < sees[t])
#pragma unroll
                            for(int b = 0; b < kBlk; ++b)
                                if(b * 32 / G == grp) o[t][b] += NAN;
                }
        }

        const bool ends = here.step + 1 == here.steps;
        if(ends || left == 1) {
#pragma unroll
            for(int t = 0; t < T; ++t) finish(t, ends);
            __syncthreads();
        }
        if(left == 1) break;
        here      = next;
        next      = after;
        page_next = page_after;
        if(ends) { // the next unit
            from_start = true;
            begin_unit();
            fetch_queries(here);
            keep_queries();
        }
    }
    if(runs.cut && threadIdx.x == 0) runs.tasks[run] = tasks;
}

// Blocks for the sequences of more than 32 rows a key head (MORE: the caller expects some), two
// times 32 rows a unit, which unpacks its codes once for both, then for those of up to 32.
template <int D, int G, bool MORE>
__global__ void __launch_bounds__(kThreads, 2)
    attention_kv4_chunks_kernel(CacheView c, ChunkArgs a, Runs few, Runs more,
                                const uint8_t* others, uint32_t pages)
{
    // the waves' values (at a unit's end halves of their results), then the queries
    __shared__ alignas(256) uint8_t lds[kWaves * kKeys * D * 2 + (MORE ? 64 : 32) * D * 2];
    __shared__ float                ml[kWaves * 32 * 2];
    const Ways     ways{others, a.heads / c.kv_heads, a.table_cols << c.page_shift, MORE};
    if(!MORE || blockIdx.x >= more.count)
        chunks_run<D, G, 1>(c, a, few, ways, blockIdx.x - (MORE ? more.count : 0), pages, lds, ml);
    else if constexpr(MORE)
        chunks_run<D, G, 2>(c, a, more, ways, blockIdx.x, pages, lds, ml);
}

// ---- the join ---------------------------------------------------------------------------
// What the cut units of one kernel's runs look like: `members` blocks a run (else 1), each of
// which has `rows` rows of a unit: of `heads` query heads and then of neighbouring rows.
struct JoinSet {
    Runs     runs;
    uint32_t members, heads, rows;
    uint32_t per;     // query heads that a sequence's rows go round
    uint32_t first;   // entry of its first run
    float    unit;    // of the sums of p v
    bool     natural; // their channels in order, else in the codes' order
};
constexpr uint32_t kJoinMost = 2 * kBlocks + kUnpackedBlocks; // entries at the most

struct JoinSets {
    JoinSet         set[3];
    const uint32_t* tasks; // of each entry
    uint32_t        entries;
};

// Joins the partials of the cut units: the second slot of the run a unit begins in, then the
// first ones of the runs after it.  Every block adds up by itself how many tasks the runs'
// cut units make, and takes its share of them.  Lanes are 8 channels each.  Of few partials a
// task is 32 (64) rows, two a group of lanes; of many one row, of which each group takes every
// 16th (32nd) partial, and the groups are added up, always in the same order.  Bound by the
// partials' latency (24 sequences of 5 tokens 9 us) and, behind long chunks, by memory (15 to
// 20 us for up to 100 MB).
template <int D>
__global__ void __launch_bounds__(kThreads, 4)
    attention_kv4_chunks_join_kernel(ChunkArgs a, JoinSets j)
{
    constexpr uint32_t kLanes = D / 8, kGroups = kThreads / kLanes;
    constexpr uint32_t kEach = (kJoinMost + kThreads - 1) / kThreads;
    static_assert(kJoinRows<D> == 2 * kGroups, "two rows a group");
    __shared__ uint32_t  before[kEach * kThreads], part[kWaves];
    __shared__ float     weights[kGroups][2];
    __shared__ alignas(16) float sums[kGroups][kLanes][8];
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const uint32_t ch = threadIdx.x % kLanes, group = threadIdx.x / kLanes;

    // ---- how many tasks come before each entry -----------------------------------------
    uint32_t mine[kEach], all = 0;
#pragma unroll
    for(uint32_t i = 0; i < kEach; ++i) {
        const uint32_t e = threadIdx.x * kEach + i;
        mine[i]          = e < j.entries ? j.tasks[e] : 0;
    }
#pragma unroll
    for(uint32_t i = 0; i < kEach; ++i) all += mine[i];
    const uint32_t s = lanes_sum(all);
    if(lane == kWave - 1) part[wave] = s;
    __syncthreads();
    uint32_t at = s - all, total = 0;
#pragma unroll
    for(uint32_t w = 0; w < kWaves; ++w) {
        if(w < wave) at += part[w];
        total += part[w];
    }
#pragma unroll
    for(uint32_t i = 0; i < kEach; ++i) {
        before[threadIdx.x * kEach + i] = at;
        at += mine[i];
    }
    __syncthreads();

    for(uint32_t task = blockIdx.x; task < total; task += gridDim.x) {
        uint32_t lo = 0, hi = kEach * kThreads; // before[lo] <= task < before[hi]
        while(hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if(before[mid] <= task)
                lo = mid;
            else
                hi = mid;
        }
        lo                     = __builtin_amdgcn_readfirstlane(lo);
        const uint32_t which   = lo < j.set[1].first ? 0 : lo < j.set[2].first ? 1 : 2;
        const JoinSet& set     = j.set[which];
        const uint32_t run     = (lo - set.first) / set.members;
        const uint32_t member  = (lo - set.first) % set.members;
        const Piece    p       = set.runs.cut[run];
        const uint32_t row0    = p.row0 + member / set.heads * set.rows;
        const uint32_t live    = min(set.rows, p.rows - row0);
        const uint32_t n       = p.last - run; // partials
        const bool     many    = join_many(n, live);
        const uint32_t of      = task - before[lo];
        uint32_t       in[2]   = {many ? of : of * kJoinRows<D> + group, 0};
        in[1]                  = many ? live : in[0] + kGroups; // its rows of the member's
        float      m[2] = {-INFINITY, -INFINITY}, l[2] = {}, sum[2][8] = {};
        const auto take = [&](int y, float mi, float li, const float* v) { // -inf: no key seen
            const float now = fmaxf(m[y], mi);
            const float al  = m[y] == now ? 1.f : __builtin_amdgcn_exp2f(m[y] - now);
            const float w
                = mi == -INFINITY ? 0.f : mi == now ? 1.f : __builtin_amdgcn_exp2f(mi - now);
            m[y] = now;
            l[y] = fmaf(l[y], al, mi == -INFINITY ? li : w * li); // 0, or NaN
            if(mi != -INFINITY)
#pragma unroll
                for(int z = 0; z < 8; ++z) sum[y][z] = fmaf(sum[y][z], al, w * v[z]);
        };
        const uint32_t step = many ? kGroups : 1;
        const auto     pass = [&](uint32_t i0, auto ahead) { // so many partials of a row
            constexpr int kAhead = decltype(ahead)::value;
            v2f ml[kAhead][2];
            v4f v[kAhead][2][2];
#pragma unroll
            for(int x = 0; x < kAhead; ++x)
#pragma unroll
                for(int y = 0; y < 2; ++y) {
                    const uint32_t i = min(i0 + x * step, n - 1);
                    const size_t   slot
                        = ((size_t)(2 * (run + i) + (i == 0 ? 1 : 0)) * set.members + member)
                              * set.rows
                          + min(in[y], live - 1);
                    const v4f* from = reinterpret_cast<const v4f*>(set.runs.o + slot * D + ch * 8);
                    ml[x][y]   = *reinterpret_cast<const v2f*>(set.runs.ml + slot * 2);
                    v[x][y][0] = from[0];
                    v[x][y][1] = from[1];
                }
#pragma unroll
            for(int x = 0; x < kAhead; ++x) {
                if(i0 + x * step >= n) continue;
#pragma unroll
                for(int y = 0; y < 2; ++y) {
                    const v4f   u0 = v[x][y][0], u1 = v[x][y][1];
                    const float w[8] = {u0[0], u0[1], u0[2], u0[3], u1[0], u1[1], u1[2], u1[3]};
                    take(y, ml[x][y][0], ml[x][y][1], w);
                }
            }
        };
        if(many)
            for(uint32_t i0 = group; i0 < n; i0 += 4 * kGroups)
                pass(i0, std::integral_constant<int, 4>());
        else
            for(uint32_t i0 = 0; i0 < n; i0 += 2) pass(i0, std::integral_constant<int, 2>());
        if(many) { // the groups' parts, one after the other
            __syncthreads();
            if(ch == 0) {
                weights[group][0] = m[0];
                weights[group][1] = l[0];
            }
#pragma unroll
            for(int z = 0; z < 8; z += 4)
                *reinterpret_cast<v4f*>(&sums[group][ch][z])
                    = v4f{sum[0][z], sum[0][z + 1], sum[0][z + 2], sum[0][z + 3]};
            __syncthreads();
            if(group == 0)
                for(uint32_t g = 1; g < kGroups; ++g)
                    take(0, weights[g][0], weights[g][1], sums[g][ch]);
            else
                in[0] = live;
        }
#pragma unroll
        for(int y = 0; y < 2; ++y) {
            if(in[y] >= live) continue;
            const float inv = l[y] != 0.f ? set.unit / l[y] : 0.f;
            float       r[8];
#pragma unroll
            for(int z = 0; z < 8; ++z) r[z] = sum[y][z] * inv;
            const uint32_t row = row0 + in[y];
            // the codes' order: places 0 .. 7 are channels 0 4 1 5 2 6 3 7
            const v4i w
                = set.natural
                      ? v4i{(int)finite_halves(r[0], r[1]), (int)finite_halves(r[2], r[3]),
                            (int)finite_halves(r[4], r[5]), (int)finite_halves(r[6], r[7])}
                      : v4i{(int)finite_halves(r[0], r[2]), (int)finite_halves(r[4], r[6]),
                            (int)finite_halves(r[1], r[3]), (int)finite_halves(r[5], r[7])};
            *reinterpret_cast<v4i*>(a.out + (size_t)(p.token + row / set.per) * a.ldo
                                    + (size_t)(p.head + row % set.per + member % set.heads) * D
                                    + ch * 8)
                = w;
        }
    }
}

// Runs of a launch: no more than steps at the most.
uint32_t run_count(uint64_t tiles, uint32_t kv_heads, uint32_t max_len)
{
    return (uint32_t)std::min<uint64_t>(kBlocks, tiles * kv_heads * steps_of(max_len));
}

// Where everything lies in the workspace: the partials of this file's kernel, then what the
// other one uses.
struct Layout {
    uint32_t       few, more;  // runs
    size_t         at[2][3];   // offsets of their sums, (maximum, sum) pairs, pieces
    size_t         tasks, other, bytes;
    UnpackedLayout u;
};

Layout layout(const w8a8_kv4_cache& c, uint32_t seqs, uint32_t tokens, uint32_t heads,
              uint32_t table_cols, uint32_t max_new)
{
    Layout         w{};
    const uint32_t max_len = table_cols * c.page_size, per = heads / c.kv_heads;
    const uint32_t most    = std::min(seqs, tokens); // sequences with new tokens
    w.few                  = run_count(most, c.kv_heads, max_len);
    if((uint64_t)std::min(max_new, tokens) * per > 32)
        w.more = run_count((uint64_t)tokens * per / 64 + most, c.kv_heads, max_len);
    size_t     at   = 0;
    const auto room = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    w.u = unpacked_layout(c, seqs, tokens, heads, table_cols, max_new);
    if(steps_of(max_len) > 1 || w.u.bytes != 0) { // else no unit is cut
        w.tasks = room(kJoinMost * 4);
        for(int i = 0; i < 2; ++i) {
            const size_t runs = i == 0 ? w.few : w.more, rows = runs * 2 * (i == 0 ? 32 : 64);
            w.at[i][0]        = room(rows * c.head_dim * 4);
            w.at[i][1]        = room(rows * 8);
            w.at[i][2]        = room(runs * sizeof(Piece));
        }
    }
    w.other = at;
    w.bytes = at + w.u.bytes;
    return w;
}

} // namespace

size_t attention_kv4_chunks_workspace_bytes(const w8a8_kv4_cache& c, uint32_t seqs,
                                            uint32_t tokens, uint32_t heads, uint32_t table_cols,
                                            uint32_t max_new)
{
    if(seqs == 0 || tokens == 0) return 0;
    return layout(c, seqs, tokens, heads, table_cols, max_new == 0 ? tokens : max_new).bytes;
}

hipError_t launch_attention_kv4_chunks(const w8a8_kv4_cache& c, const ChunkArgs& a,
                                       hipStream_t stream)
{
    const Layout w  = layout(c, a.seqs, a.tokens, a.heads, a.table_cols, a.max_new);
    auto*        ws = static_cast<uint8_t*>(a.ws);
    const bool     cut   = w.other != 0;
    const uint32_t per   = a.heads / c.kv_heads;
    auto*          tasks = reinterpret_cast<uint32_t*>(ws + w.tasks);
    Runs           runs[2]{};
    for(int i = 0; i < 2; ++i) {
        runs[i].count = i == 0 ? w.few : w.more;
        if(cut) {
            runs[i].o     = reinterpret_cast<float*>(ws + w.at[i][0]);
            runs[i].ml    = reinterpret_cast<float*>(ws + w.at[i][1]);
            runs[i].cut   = reinterpret_cast<Piece*>(ws + w.at[i][2]);
            runs[i].tasks = tasks + i * w.few;
        }
    }
    const uint32_t both = w.few + w.more;
    JoinSets       sets{{{runs[0], 1, 1, 32, per, 0, 2.f, false},
                   {runs[1], 1, 1, 64, per, w.few, 2.f, false},
                   {{}, 1, 1, 1, 1, both, 1.f, true}},
                  tasks,
                  both};
    const uint8_t* others = nullptr;
    if(w.u.bytes != 0) {
        const Runs r = unpacked_runs(w.u, ws + w.other, tasks + both);
        launch_unpacked(c, a, w.u, r, ws + w.other, stream);
        others      = ws + w.other + w.u.flags;
        sets.set[2] = {r, w.u.members, w.u.heads, 128, 1, both, 1.f, true};
        sets.entries += w.u.runs * w.u.members;
    }
    // a task is at least a row, and mostly more
    const uint32_t joins = (uint32_t)std::min<uint64_t>((uint64_t)a.tokens * a.heads, 1024);
    with_widths(c, [&](auto d, auto g) {
        const auto kernel = w.more != 0 ? attention_kv4_chunks_kernel<d(), g(), true>
                                        : attention_kv4_chunks_kernel<d(), g(), false>;
        kernel<<<w.few + w.more, kThreads, 0, stream>>>(view(c), a, runs[0], runs[1], others,
                                                       c.pages);
        if(cut)
            attention_kv4_chunks_join_kernel<d()><<<joins, kThreads, 0, stream>>>(a, sets);
    });
    return hipGetLastError();
}

} // namespace w8a8
