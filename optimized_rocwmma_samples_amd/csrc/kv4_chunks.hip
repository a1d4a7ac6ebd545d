// kv4_chunks.hip -- attention of several new tokens per sequence over the paged 4-bit
// cache, for gfx950.
//
//   out[t, h] = sum_j p[j] v[j],  p = softmax of scale * (q[t, h] . k[j]) over the tokens j of
//   t's sequence up to t itself; the rows of q are the sequence's last tokens.
//
// The rows of a unit of work are the (token, query head) pairs of one key head, 32 at a
// time: row r is token r / per, head r % per, per query heads sharing the key head.  Units
// are walked in steps of 128 keys, 32 a wave.  All units' steps lie in one line, which is
// cut into as many equal runs as there are blocks; what a cut leaves of a unit is written as
// partials (sum of p v, maximum and sum of p of each row) and joined by a second launch.
//   * S^T = K Q^T with v_mfma_f32_32x32x16_f16: srcA rows are keys, and a lane's operand is 8
//     channels of one key, which is a dword of its codes: unpacked, scaled and used where
//     it was loaded.
//   * The scores of one query row lie in a lane (and lane ^ 32), so softmax stays there, and
//     the probabilities are the srcB operand of O^T += V^T P^T as they are.
//   * V^T's rows are channels: a wave unpacks its 32 rows of values into a tile of its own in
//     LDS and reads it transposed with ds_read_b64_tr_b16.  Nothing waits for other waves
//     until the unit ends.
// A code n becomes 1024 + n by two bit operations a pair, n - 8 and then offset + scale *
// (n - 8), rounded once: half of what kv4_load gives, since a group that reaches the ends of
// fp16 may pass them by half a step (the halves go into the scale of the scores and of the
// result).
#include "kv4_chunks.hpp"

#include <algorithm>

namespace w8a8 {
namespace {

typedef float  v2f __attribute__((ext_vector_type(2)));
typedef float  v16f __attribute__((ext_vector_type(16)));
typedef __fp16 v4fp16 __attribute__((ext_vector_type(4)));

typedef __attribute__((address_space(3))) v4fp16 lds_v4h_t;
typedef __attribute__((address_space(3))) v4i    lds_v4i_t;
typedef __attribute__((address_space(3))) v4f    lds_v4f_t;

constexpr int      kWaves   = 4;
constexpr int      kThreads = kWaves * kWave;
constexpr int      kKeys    = 32;              // a wave's a step
constexpr int      kStep    = kWaves * kKeys;  // keys of a step
constexpr uint32_t kBlocks  = 512;             // two a CU

__host__ __device__ inline uint32_t steps_of(uint32_t len)
{
    return len == 0 ? 1u : (len + kStep - 1) / kStep; // a sequence of no tokens is written too
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

__device__ __forceinline__ float max3(float a, float b, float c)
{
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

__device__ __forceinline__ bool finite_pair(uint32_t w)
{
    return (w & 0x7C00u) != 0x7C00u && (w & 0x7C000000u) != 0x7C000000u;
}

// The 8 codes of a dword as fp16 values offset + scale * (n - 8), in the order 0 4 1 5 2 6 3 7;
// `pair` is (scale, offset).
struct Unpack {
    uint32_t mask, big;
    __device__ Unpack()
    {
        asm volatile("v_mov_b32 %0, 0x000f000f" : "=v"(mask));
        asm volatile("v_mov_b32 %0, 0x64006400" : "=v"(big)); // 1024, whose last bit is 1
    }
    __device__ v8h operator()(uint32_t w, v2h pair) const
    {
        const v2h middle = {(_Float16)1032.f, (_Float16)1032.f};
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

__device__ __forceinline__ v2h halved(int32_t pair)
{
    return __builtin_bit_cast(v2h, pair) * v2h{(_Float16)0.5f, (_Float16)0.5f};
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

template <int D, int G, int T>
__device__ __forceinline__ void chunks_run(const CacheView& c, const ChunkArgs& a, const Runs& runs,
                                           const uint8_t* others, uint32_t pages,
                                           uint8_t* lds, float* lds_ml)
{
    using R = Raw<D, G>;
    constexpr int  kSteps = D / 16, kBlk = D / 32; // products along the channels; result blocks
    constexpr int  kTile = kKeys * D * 2;          // bytes of a wave's values
    constexpr uint32_t kRows = 32 * T;             // rows of a unit
    const int      wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int      lane = threadIdx.x % kWave, col = lane % 32, half = lane / 32;
    const uint32_t run = blockIdx.x;
    const uint32_t per = a.heads / c.kv_heads, most = a.table_cols << c.page_shift;
    // LDS: the waves' values (at a unit's end two waves' results), then the queries
    const uint32_t lds0 = (uint32_t)(uintptr_t)lds, tile = lds0 + wave * kTile;
    const uint32_t qat = lds0 + kWaves * kTile + lane * 16;
    auto           chunk_at = [&](uint32_t i) { // without rows where they go another way
        Chunk x = chunk_of(a, i, most);
        if(others != nullptr && others[i] != 0) x.fresh = 0;
        if((x.fresh * per > 32) != (T > 1)) x.fresh = 0;
        return x;
    };
    auto           tiles_of = [&](const Chunk& s) { return (s.fresh * per + kRows - 1) / kRows; };

    // ---- the block's run ---------------------------------------------------------------
    // (in 64 bits: starts that do not ascend may count rows many times)
    auto scan = [&](uint32_t i0, uint32_t& n, uint64_t& s) { // 64 sequences' steps
        const uint32_t i = i0 + lane;
        n                = 0;
        if(i < a.seqs) {
            const Chunk x = chunk_at(i);
            n             = tiles_of(x) * c.kv_heads * steps_of(x.len);
        }
        s = n;
#pragma unroll
        for(int d = 1; d < kWave; d <<= 1) {
            const uint64_t o = __shfl_up((unsigned long long)s, d, kWave);
            if(lane >= d) s += o;
        }
        return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)s, kWave - 1)
               | (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(s >> 32), kWave - 1)
                     << 32;
    };
    uint32_t n;
    uint64_t s, all = 0;
    for(uint32_t i = 0; i < a.seqs; i += kWave) all += scan(i, n, s);
    if(all > 0x7FFFFFFFull) all = 0;
    const uint32_t q = (uint32_t)all / runs.count, r = (uint32_t)all % runs.count;
    uint32_t       at = run * q + min(run, r), left = q + (run < r ? 1 : 0);
    if(runs.cut && threadIdx.x == 0) runs.cut[run].last = 0;
    if(left == 0) return;
    const uint32_t end = at + left;
    Place          here{};
    for(uint32_t i = 0; i < a.seqs; i += kWave) {
        const uint32_t sum = (uint32_t)scan(i, n, s);
        if(at < sum) {
            const int f = __builtin_ctzll(__ballot(s > at));
            at -= (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)s, f)
                  - (uint32_t)__builtin_amdgcn_readlane((int)n, f);
            here.seq = i + f;
            break;
        }
        at -= sum;
    }
    auto enter = [&](Place& p) { // the sequence p.seq
        p.c     = chunk_at(p.seq);
        p.steps = steps_of(p.c.len);
        p.tiles = tiles_of(p.c);
    };
    enter(here);
    here.unit = at / here.steps;
    here.step = at % here.steps;
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
    auto page_at = [&](const Place& p) { // of the lane's key
        const uint32_t t    = p.step * kStep + wave * kKeys + col;
        int32_t        page = -1;
        if(t < p.c.len) {
            page = a.table[(size_t)p.seq * a.table_ld + (t >> c.page_shift)];
            if(page < 0 || (uint32_t)page >= pages) page = -1;
        }
        return page;
    };
    auto fetch = [&](R& x, const Place& p, int32_t page) {
        x.ok             = page >= 0; // without one page 0's rows are read, and masked
        const size_t row = cache_row(c, page >= 0 ? page : 0, p.unit / p.tiles,
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
    const auto queries = [&](const Place& p) {
        const uint32_t row0 = p.unit % p.tiles * kRows, rows = p.c.fresh * per;
        auto           seen = [&](uint32_t row) {
            return (uint32_t)max((int32_t)(p.c.len + row / per + 1 - p.c.fresh), 0);
        };
        constexpr int kOrder[8] = {0, 4, 1, 5, 2, 6, 3, 7};
        least                   = seen(row0);
#pragma unroll
        for(int t = 0; t < T; ++t) {
            const uint32_t row = min(row0 + 32 * t + col, rows - 1);
            sees[t]            = seen(row);
            const uint16_t* from = a.q + (size_t)(p.c.begin + row / per) * a.ldq
                                   + (size_t)(p.unit / p.tiles * per + row % per) * D + 8 * half;
#pragma unroll
            for(int st = wave; st < kSteps; st += kWaves) {
                const v8h v = *reinterpret_cast<const v8h*>(from + 16 * st);
                v8h       u;
#pragma unroll
                for(int e = 0; e < 8; ++e) u[e] = v[kOrder[e]];
                *(lds_v4i_t*)(uintptr_t)(qat + (t * kSteps + st) * kWave * 16)
                    = __builtin_bit_cast(v4i, u);
            }
        }
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
    Place next = here;
    {
        const int32_t page = page_at(here);
        queries(here);
        fetch(x, here, page);
    }
    int32_t page_next = -1;
    if(left > 1) {
        advance(next);
        page_next = page_at(next);
    }
    __syncthreads(); // the queries are there

    // The waves' results of 32 rows joined and written, at the unit's end or the run's.
    auto finish = [&](const int t, const Place& now, bool ends) {
        const v2f ls = both_halves(l[t]);
        const float lw = ls[0] + ls[1];
        if(half == 0) {
            lds_ml[(wave * 32 + col) * 2]     = m[t];
            lds_ml[(wave * 32 + col) * 2 + 1] = lw;
        }
        __syncthreads();
        float common = -INFINITY, sum = 0.f;
#pragma unroll
        for(int w = 0; w < kWaves; ++w) common = fmaxf(common, lds_ml[(w * 32 + col) * 2]);
        auto weight = [&](float mw) {
            return mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mw - common) * c2);
        };
#pragma unroll
        for(int w = 0; w < kWaves; ++w)
            sum = fmaf(weight(lds_ml[(w * 32 + col) * 2]), lds_ml[(w * 32 + col) * 2 + 1], sum);
        const float mine = weight(m[t]);
#pragma unroll
        for(int b = 0; b < kBlk; ++b) o[t][b] *= mine;
        // the waves' results added up: 2 and 3 to 0 and 1, then 1 to 0
#pragma unroll
        for(int d = 2; d > 0; d /= 2) {
            const uint32_t buf = lds0 + (wave % d) * (kBlk * 16 * kWave * 4) + lane * 16;
            if(wave >= d && wave < 2 * d)
#pragma unroll
                for(int b = 0; b < kBlk; ++b)
#pragma unroll
                    for(int i = 0; i < 16; i += 4)
                        *(lds_v4f_t*)(uintptr_t)(buf + (b * 4 + i / 4) * kWave * 16)
                            = v4f{o[t][b][i], o[t][b][i + 1], o[t][b][i + 2], o[t][b][i + 3]};
            __syncthreads();
            if(wave < d)
#pragma unroll
                for(int b = 0; b < kBlk; ++b)
#pragma unroll
                    for(int i = 0; i < 16; i += 4) {
                        const v4f u
                            = *(lds_v4f_t*)(uintptr_t)(buf + (b * 4 + i / 4) * kWave * 16);
#pragma unroll
                        for(int e = 0; e < 4; ++e) o[t][b][i + e] += u[e];
                    }
            __syncthreads();
        }
        if(wave != 0) return;
        const uint32_t row0 = now.unit % now.tiles * kRows + 32 * t, rows = now.c.fresh * per;
        const uint32_t row = row0 + col, head0 = now.unit / now.tiles * per;
        if(ends && from_start) {
            const float inv = sum != 0.f ? 2.f / sum : 0.f;
            uint16_t*   out = a.out + (size_t)(now.c.begin + row / per) * a.ldo
                            + (size_t)(head0 + row % per) * D + 4 * half;
#pragma unroll
            for(int b = 0; b < kBlk; ++b)
#pragma unroll
                for(int i = 0; i < 16; i += 4) {
                    // this half has channels 0 1, 4 5 (2 3, 6 7) of a chunk of 8
                    const auto w = __builtin_amdgcn_permlane32_swap(
                        finite_halves(o[t][b][i] * inv, o[t][b][i + 2] * inv),
                        finite_halves(o[t][b][i + 1] * inv, o[t][b][i + 3] * inv), false, false);
                    if(row < rows)
                        *reinterpret_cast<v2i*>(out + 32 * b + 8 * (i / 4))
                            = v2i{(int)w[0], (int)w[1]};
                }
        } else if(row < rows) {
            const size_t slot = (size_t)(2 * run + (from_start ? 1 : 0)) * kRows + 32 * t + col;
#pragma unroll
            for(int b = 0; b < kBlk; ++b)
#pragma unroll
                for(int i = 0; i < 16; i += 4)
                    *reinterpret_cast<v4f*>(runs.o + slot * D + 32 * b + 2 * i + 4 * half)
                        = v4f{o[t][b][i], o[t][b][i + 1], o[t][b][i + 2], o[t][b][i + 3]};
            if(half == 0) *reinterpret_cast<v2f*>(runs.ml + slot * 2) = v2f{common * c2, sum};
        }
        if(t == 0 && !ends && from_start && lane == 0) { // goes on behind the run: up to which
            const uint32_t last = end - 1 + (now.steps - 1 - now.step); // its last step
            runs.cut[run]       = {(last < r * (q + 1) ? last / (q + 1)
                                                       : r + (last - r * (q + 1)) / q) + 1,
                             now.c.begin, row0, rows, head0, {}};
        }
    };

    for(; left > 0; --left) {
        const Place    now  = here;
        const uint32_t key0 = now.step * kStep + wave * kKeys;
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
            vs[g] = halved(x.vs[g]);
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
            const v8h k = unpack((uint32_t)x.k[st % 2][st / 2], halved(x.ks[st / 2 * 32 / G]));
#pragma unroll
            for(int t = 0; t < T; ++t)
                sc[t] = mfma(k,
                             __builtin_bit_cast(v8h, *(lds_v4i_t*)(uintptr_t)(
                                                         qat + (t * kSteps + st) * kWave * 16)),
                             sc[t]);
        }
        if(left > 1) { // the next step's loads, over the rest of this one
            const int32_t page = page_next;
            here               = next;
            if(left > 2) {
                advance(next);
                page_next = page_at(next);
            }
            fetch(x, here, page);
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
                    const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[t][st * 8 + i + 1], c2, -mc[t]));
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

        const bool ends = now.step + 1 == now.steps;
        if(!ends && left > 1) continue;
#pragma unroll
        for(int t = 0; t < T; ++t) finish(t, now, ends);
        if(left > 1) { // the next unit
            from_start = true;
            begin_unit();
            queries(here);
            __syncthreads();
        }
    }
}

// Sequences of up to 32 rows a key head, then (MORE: there may be any) those of more, two
// times 32 rows a unit, which unpacks its codes once for both.
template <int D, int G, bool MORE>
__global__ void __launch_bounds__(kThreads, 2)
    attention_kv4_chunks_kernel(CacheView c, ChunkArgs a, Runs few, Runs more,
                                const uint8_t* others, uint32_t pages)
{
    __shared__ alignas(256) uint8_t lds[kWaves * kKeys * D * 2 + (MORE ? 64 : 32) * D * 2];
    __shared__ float                ml[kWaves * 32 * 2];
    if(blockIdx.x < few.count) chunks_run<D, G, 1>(c, a, few, others, pages, lds, ml);
    if constexpr(MORE) {
        __syncthreads();
        if(blockIdx.x < more.count) chunks_run<D, G, 2>(c, a, more, others, pages, lds, ml);
    }
}

// Joins the partials of the cut units: the second slot of the run a unit begins in, then the
// first ones of the runs after it.  A wave has 4 rows, lanes being 8 channels each.  Few
// partials are taken by all four rows' lanes at once, each its own; of many a row at a time,
// its lanes each every fourth, then the four are added up, in the same order always.
template <int D>
__global__ void __launch_bounds__(kThreads)
    attention_kv4_chunks_join_kernel(ChunkArgs a, Runs few, Runs more, uint32_t per)
{
    constexpr uint32_t kLanes = D / 8, kWays = kWave / kLanes, kMany = 16;
    const uint32_t     lane = threadIdx.x % kWave, ch = lane % kLanes, way = lane / kLanes;
    const uint32_t     first = few.count * (32 / kWays), all = first + more.count * (64 / kWays);
    for(uint32_t task = blockIdx.x * kWaves + threadIdx.x / kWave; task < all;
        task += gridDim.x * kWaves) {
        const bool     is_few = task < first;
        const Runs&    runs   = is_few ? few : more;
        const uint32_t rows = is_few ? 32 : 64, of = is_few ? task : task - first;
        const uint32_t run  = __builtin_amdgcn_readfirstlane(of / (rows / kWays));
        const uint32_t in0  = of % (rows / kWays) * kWays;
        const Piece    u    = runs.cut[run];
        if(u.last == 0 || u.row0 + in0 >= u.rows) continue;
        const uint32_t n = u.last - run; // partials
        float          m, l, sum[8];
        auto           clear = [&] {
            m = -INFINITY;
            l = 0.f;
#pragma unroll
            for(int y = 0; y < 8; ++y) sum[y] = 0.f;
        };
        auto take = [&](float mi, float li, const float* v) { // -inf: no key seen
            const float now = fmaxf(m, mi);
            const float al  = m == now ? 1.f : __builtin_amdgcn_exp2f(m - now);
            const float e   = mi == -INFINITY ? 0.f : mi == now ? 1.f : __builtin_amdgcn_exp2f(mi - now);
            m               = now;
            l               = fmaf(l, al, mi == -INFINITY ? li : e * li); // 0, or NaN
            if(e != 0.f)
#pragma unroll
                for(int y = 0; y < 8; ++y) sum[y] = fmaf(sum[y], al, e * v[y]);
        };
        auto add = [&](uint32_t i, uint32_t in) {
            const size_t slot = (size_t)(2 * (run + i) + (i == 0 ? 1 : 0)) * rows + in;
            const v2f    ml   = *reinterpret_cast<const v2f*>(runs.ml + slot * 2);
            const v4f*   v    = reinterpret_cast<const v4f*>(runs.o + slot * D + ch * 8);
            const v4f    v0 = v[0], v1 = v[1];
            const float  both[8] = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
            take(ml[0], ml[1], both);
        };
        auto write = [&](uint32_t in) {
            const uint32_t row = u.row0 + in;
            const float    inv = l != 0.f ? 2.f / l : 0.f;
#pragma unroll
            for(int y = 0; y < 8; ++y) sum[y] *= inv;
            // places 0 .. 7 are channels 0 4 1 5 2 6 3 7
            if(row < u.rows)
                *reinterpret_cast<v4i*>(a.out + (size_t)(u.token + row / per) * a.ldo
                                        + (size_t)(u.head + row % per) * D + ch * 8)
                    = v4i{(int)finite_halves(sum[0], sum[2]), (int)finite_halves(sum[4], sum[6]),
                          (int)finite_halves(sum[1], sum[3]), (int)finite_halves(sum[5], sum[7])};
        };
        if(n <= kMany) {
            clear();
            const uint32_t in = min(in0 + way, u.rows - 1 - u.row0);
            for(uint32_t i = 0; i < n; ++i) add(i, in);
            write(in0 + way);
            continue;
        }
        for(uint32_t y = 0; y < kWays && u.row0 + in0 + y < u.rows; ++y) {
            clear();
            for(uint32_t i = way; i < n; i += kWays) add(i, in0 + y);
#pragma unroll
            for(uint32_t d = kLanes; d < kWave; d <<= 1) {
                const float mo = __shfl_xor(m, d, kWave), lo = __shfl_xor(l, d, kWave);
                float       vo[8];
#pragma unroll
                for(int z = 0; z < 8; ++z) vo[z] = __shfl_xor(sum[z], d, kWave);
                take(mo, lo, vo);
            }
            if(way == 0) write(in0 + y);
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
    size_t         other, bytes;
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
    if(steps_of(max_len) > 1) // else no unit is cut
        for(int i = 0; i < 2; ++i) {
            const size_t runs = i == 0 ? w.few : w.more, rows = runs * 2 * (i == 0 ? 32 : 64);
            w.at[i][0]        = room(rows * c.head_dim * 4);
            w.at[i][1]        = room(rows * 8);
            w.at[i][2]        = room(runs * sizeof(Piece));
        }
    w.other = at;
    w.u     = unpacked_layout(c, seqs, tokens, heads, table_cols, max_new);
    w.bytes = w.other + w.u.bytes;
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
    const bool   cut = w.other != 0;
    Runs         runs[2]{};
    for(int i = 0; i < 2; ++i) {
        runs[i].count = i == 0 ? w.few : w.more;
        if(cut) {
            runs[i].o   = reinterpret_cast<float*>(ws + w.at[i][0]);
            runs[i].ml  = reinterpret_cast<float*>(ws + w.at[i][1]);
            runs[i].cut = reinterpret_cast<Piece*>(ws + w.at[i][2]);
        }
    }
    const uint8_t* others = nullptr;
    if(w.u.bytes != 0) {
        launch_unpacked(c, a, w.u, ws + w.other, stream);
        others = ws + w.other + w.u.flags;
    }
    with_widths(c, [&](auto d, auto g) {
        const auto kernel = w.more != 0 ? attention_kv4_chunks_kernel<d(), g(), true>
                                        : attention_kv4_chunks_kernel<d(), g(), false>;
        kernel<<<std::max(w.few, w.more), kThreads, 0, stream>>>(view(c), a, runs[0], runs[1],
                                                                others, c.pages);
        if(cut) {
            const uint32_t tasks = (w.few * 32 + w.more * 64) / (kWave / (d() / 8));
            attention_kv4_chunks_join_kernel<d()>
                <<<std::min((tasks + kWaves - 1) / kWaves, 1024u), kThreads, 0, stream>>>(
                    a, runs[0], runs[1], a.heads / c.kv_heads);
        }
    });
    return hipGetLastError();
}

} // namespace w8a8
