// kv4_pages.hip -- the pages of the 4-bit cache for gfx950: handing them out and taking
// them back, a key for each page, and the pages that suit a query.
#include "kv4_device.hpp"

#include <algorithm>
#include <cmath>

namespace w8a8 {
namespace {

// ---------------------------------------------------------------------------
// Pages handed out and taken back.
//
// Where a sequence's tokens and pages go follows from two running sums over the sequences
// (new tokens, pages needed).  Every block computes them by itself, 1024 sequences at a
// time, so that none waits for another, and then takes its share of the tokens and pages,
// finding each one's sequence by halving among the 1024 sums in LDS.  The lengths and the
// count are written by the first block, or, with more than one, by a second launch of one
// where the caller has them written over the lengths and the count that every block reads.
//
// Bound by latency: lengths, sums with two barriers, a page number, a write.  MI355X: a step of
// 256 sequences 5.8 us in one block, 48 prompts of some 32000 rows 6.7 in 32; 24 sequences
// trimmed 3.8, 512 of 262144 columns 6.  A second launch costs a call 3 us.
// ---------------------------------------------------------------------------
constexpr int kSeqs = 1024; // threads of a block, and sequences a step

// Running sums over a block's threads, without the own value; `all` is the sum of all.
__device__ __forceinline__ uint64_t block_sum(uint64_t v, uint64_t* part, uint64_t& all)
{
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    uint64_t  s = v;
#pragma unroll
    for(int d = 1; d < kWave; d <<= 1) {
        const uint64_t o = __shfl_up((unsigned long long)s, d, kWave);
        if(lane >= d) s += o;
    }
    __syncthreads(); // the last step's values are read
    if(lane == kWave - 1) part[wave] = s;
    __syncthreads();
    uint64_t before = 0;
    all             = 0;
#pragma unroll
    for(int w = 0; w < kSeqs / kWave; ++w) {
        if(w < wave) before += part[w];
        all += part[w];
    }
    return before + s - v;
}

// The last of n ascending values that is not above x; the first where all are.
__device__ __forceinline__ uint32_t last_not_above(const uint32_t* v, uint32_t n, uint32_t x)
{
    uint32_t lo = 0, hi = n; // v[lo] <= x < v[hi]
    while(hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if(v[mid] <= x)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// The block's rounds of 1024 of the numbers lo .. hi - 1: which number is this thread's.
template <class F>
__device__ __forceinline__ void shares(uint32_t lo, uint32_t hi, F f)
{
    if(lo >= hi) return;
    const uint32_t first = lo / kSeqs, g = gridDim.x;
    for(uint32_t r = first + (blockIdx.x + g - first % g) % g; r <= (hi - 1) / kSeqs; r += g) {
        const uint32_t x = r * kSeqs + threadIdx.x;
        if(x >= lo && x < hi) f(x);
    }
}

__device__ __forceinline__ uint32_t clamped(int32_t v, uint32_t most)
{
    return v < 0 ? 0u : min((uint32_t)v, most);
}

template <bool PLACES, bool COMMIT>
__global__ void __launch_bounds__(kSeqs) kv4_extend_kernel(Kv4ExtendArgs a)
{
    __shared__ uint64_t part[kSeqs / kWave];
    __shared__ uint32_t begins[kSeqs], bases[kSeqs], lengths[kSeqs], taken;
    const uint32_t shift = a.page_shift, p = 1u << shift, most = a.table_cols << shift;
    const uint32_t avail = clamped(a.count[0], a.capacity);
    uint64_t       rows = 0, pages = 0; // of the sequences before
    if(threadIdx.x == 0) taken = 0;
    for(uint32_t i0 = 0; i0 < a.seqs; i0 += kSeqs) {
        const uint32_t i = i0 + threadIdx.x;
        const bool     is = i < a.seqs;
        // more than all rows is as good as that many and one
        const uint32_t n   = is ? clamped(a.fresh[i], a.tokens + 1) : 0;
        const uint32_t len = is ? clamped(a.lens[i], most) : 0;
        uint64_t       all_rows, all_pages;
        const uint64_t begin = rows + block_sum(n, part, all_rows);
        const bool     fits  = begin + n <= a.tokens && (uint64_t)len + n <= most;
        const uint32_t need  = fits ? (len + n + p - 1) / p - (len + p - 1) / p : 0;
        const uint64_t base  = pages + block_sum(need, part, all_pages);
        const bool     given = is && fits && (need == 0 || base + need <= avail);
        // (block_sum's barriers lie behind the last step's reads of these)
        begins[threadIdx.x]  = (uint32_t)min(begin, (uint64_t)a.tokens);
        bases[threadIdx.x]   = (uint32_t)base;
        lengths[threadIdx.x] = given ? len : 0xFFFFFFFFu;
        if(COMMIT && blockIdx.x == 0 && is) {
            a.starts[i] = (int32_t)min(begin, (uint64_t)a.tokens);
            if(given && need != 0) atomicMax(&taken, (uint32_t)base + need);
            a.lens_out[i] = (int32_t)(given ? len + n : len);
        }
        __syncthreads();
        if(PLACES) {
            const uint32_t in = min((uint32_t)kSeqs, a.seqs - i0);
            // the table's new columns
            shares((uint32_t)pages, (uint32_t)min(pages + all_pages, (uint64_t)avail),
                   [&](uint32_t f) {
                       const uint32_t s = last_not_above(bases, in, f), l = lengths[s];
                       if(l == 0xFFFFFFFFu) return;
                       const uint32_t col = (l + p - 1) / p + (f - bases[s]);
                       a.table[(size_t)(i0 + s) * a.table_ld + col] = a.free[avail - 1 - f];
                   });
            // the new tokens' slots
            shares((uint32_t)min(rows, (uint64_t)a.tokens),
                   (uint32_t)min(rows + all_rows, (uint64_t)a.tokens), [&](uint32_t t) {
                       const uint32_t s = last_not_above(begins, in, t), l = lengths[s];
                       int64_t        slot = -1;
                       if(l != 0xFFFFFFFFu) {
                           const uint32_t at = l + (t - begins[s]), old = (l + p - 1) / p;
                           const uint32_t col = at >> shift;
                           const int32_t  page
                               = col < old ? a.table[(size_t)(i0 + s) * a.table_ld + col]
                                           : a.free[avail - 1 - (bases[s] + col - old)];
                           slot = (int64_t)page * p + (at & (p - 1));
                           if(page < 0 || slot > 0x7FFFFFFF) slot = -1;
                       }
                       a.slots[t] = (int32_t)slot;
                   });
        }
        rows += all_rows;
        pages += all_pages;
    }
    if(PLACES) // rows behind the last sequence
        shares((uint32_t)min(rows, (uint64_t)a.tokens), a.tokens,
               [&](uint32_t t) { a.slots[t] = -1; });
    if(COMMIT && blockIdx.x == 0) {
        __syncthreads();
        if(threadIdx.x == 0) {
            a.starts[a.seqs] = (int32_t)min(rows, (uint64_t)a.tokens);
            a.count_out[0]   = (int32_t)(avail - taken);
        }
    }
}

template <bool PLACES, bool COMMIT>
__global__ void __launch_bounds__(kSeqs) kv4_trim_kernel(Kv4TrimArgs a)
{
    __shared__ uint64_t part[kSeqs / kWave];
    __shared__ uint32_t bases[kSeqs], firsts[kSeqs];
    const uint32_t shift = a.page_shift, p = 1u << shift, most = a.table_cols << shift;
    const uint32_t avail = clamped(a.count[0], a.capacity);
    auto pages_of = [&](uint32_t i, uint32_t& kept, uint32_t& first) { // that sequence i gives back
        if(i >= a.seqs) return 0u;
        const uint32_t len = clamped(a.lens[i], most);
        kept               = min(clamped(a.keep[i], most), len);
        first              = (kept + p - 1) / p;
        return (len + p - 1) / p - first;
    };
    uint32_t kept = 0, first = 0;
    uint64_t all = 0, sum, pages = 0;
    for(uint32_t i0 = 0; i0 < a.seqs; i0 += kSeqs) {
        block_sum(pages_of(i0 + threadIdx.x, kept, first), part, sum);
        all += sum;
    }
    for(uint32_t i0 = 0; i0 < a.seqs; i0 += kSeqs) {
        const uint32_t i = i0 + threadIdx.x, n = pages_of(i, kept, first);
        const uint64_t base  = pages + block_sum(n, part, sum);
        bases[threadIdx.x]  = (uint32_t)base;
        firsts[threadIdx.x] = first;
        if(COMMIT && blockIdx.x == 0 && i < a.seqs) a.lens_out[i] = (int32_t)kept;
        __syncthreads();
        if(PLACES) {
            const uint32_t in = min((uint32_t)kSeqs, a.seqs - i0);
            shares((uint32_t)pages, (uint32_t)(pages + sum), [&](uint32_t f) {
                const uint32_t s  = last_not_above(bases, in, f);
                const uint64_t to = avail + (all - 1 - f);
                if(to < a.capacity)
                    a.free[to]
                        = a.table[(size_t)(i0 + s) * a.table_ld + firsts[s] + (f - bases[s])];
            });
        }
        pages += sum;
    }
    if(COMMIT && blockIdx.x == 0) {
        if(threadIdx.x == 0) a.count_out[0] = (int32_t)min(avail + all, (uint64_t)a.capacity);
    }
}

// ---------------------------------------------------------------------------
// Page keys: the mean of the keys of a page's tokens, in 8 bits with a power of two as the
// scale.  Codes and scales of the cache are fp16 and small whole numbers, so their values
// and sums are exact in 64 bits, in any order; the quotient is rounded once, and a power of
// two adds no rounding, so page keys are the same wherever they are computed.
//
// A wave takes one key head of one page: lane = 8 channels (a dword of codes) of every
// 4th (8th) row.  Bound by the start and one read's latency: 64 rows are 16 dwords a lane,
// all on their way together.  MI355X, 8 key heads of 128: the 128 pages of 8192 tokens 6.1 us
// (5.9 MB), a step of 48 sequences 5.
// ---------------------------------------------------------------------------
constexpr int kWaveThreads = 256;

__device__ __forceinline__ double of_halves(uint32_t lo, uint32_t hi)
{
    return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}

// v and the one D lanes away, added up: D = 8, 16 or 32.
template <int D>
__device__ __forceinline__ double add_across(double v)
{
    const uint64_t u = (uint64_t)__double_as_longlong(v);
    const uint32_t lo = (uint32_t)u, hi = (uint32_t)(u >> 32);
    if constexpr(D == 32) {
        const auto l = __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
        const auto h = __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
        return of_halves(l[0], h[0]) + of_halves(l[1], h[1]);
    } else if constexpr(D == 16) {
        const auto l = __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
        const auto h = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
        return of_halves(l[0], h[0]) + of_halves(l[1], h[1]);
    } else
        return v + of_halves((uint32_t)dpp_mov_i32<kDppRowRor8>((int)lo),
                             (uint32_t)dpp_mov_i32<kDppRowRor8>((int)hi));
}

// The least e with |v| <= 127 * 2^e; kNoPower of 0.  It grows with |v|, so the largest of
// several is that of the largest value.
constexpr int kNoPower = -5000;
__device__ __forceinline__ int power_for(double v)
{
    int          e;
    const double m = frexp(fabs(v), &e);
    return v == 0.0 ? kNoPower : m <= 127.0 / 128.0 ? e - 7 : e - 6;
}

__device__ __forceinline__ int wave_max_i32(int v) { return -wave_min_i32(-v); }

template <int D, int G>
__global__ void __launch_bounds__(kWaveThreads)
    kv4_summarize_kernel(CacheView c, Kv4SummarizeArgs a, uint32_t pages)
{
    constexpr int  kLanes = D / 8, kRows = kWave / kLanes, kAhead = 16;
    const int      lane = threadIdx.x % kWave, x = lane % kLanes, r0 = lane / kLanes;
    const uint32_t unit = __builtin_amdgcn_readfirstlane(
        blockIdx.x * (kWaveThreads / kWave) + threadIdx.x / kWave);
    const uint32_t head = unit % c.kv_heads;
    uint32_t       at   = unit / c.kv_heads; // the touched page, then its place in a sequence

    // ---- whose page: 64 sequences a step ---------------------------------------------
    uint32_t seq = 0, col = 0, len = 0;
    bool     found = false;
    for(uint32_t i0 = 0; i0 < a.seqs; i0 += kWave) {
        const uint32_t i = i0 + lane;
        uint32_t       n = 0, from = 0, l = 0;
        if(i < a.seqs) {
            const uint32_t b = clamped(a.starts[i], a.tokens);
            const uint32_t e = clamped(a.starts[i + 1], a.tokens);
            const uint32_t fresh = e > b ? e - b : 0;
            l                    = clamped(a.lens[i], a.table_cols << c.page_shift);
            from                 = (l > fresh ? l - fresh : 0) >> c.page_shift;
            if(fresh != 0 && l != 0) n = ((l - 1) >> c.page_shift) + 1 - from;
        }
        const uint32_t s    = lanes_sum(n);
        const uint64_t past = __ballot(s > at);
        if(past != 0) {
            const int f = __builtin_ctzll(past);
            seq         = i0 + f;
            col   = __builtin_amdgcn_readlane(from, f)
                  + (at - (__builtin_amdgcn_readlane(s, f) - __builtin_amdgcn_readlane(n, f)));
            len   = __builtin_amdgcn_readlane(l, f);
            found = true;
            break;
        }
        at -= __builtin_amdgcn_readlane(s, kWave - 1);
    }
    if(!found) return;
    const int32_t page = a.table[(size_t)seq * a.table_ld + col];
    if(page < 0 || (uint32_t)page >= pages) return;
    const uint32_t rows = min(c.page_size, len - (col << c.page_shift));

    // ---- the sum ----------------------------------------------------------------------
    // dword x of a row of keys: channels 32 j + 8 g .. with x = g * (D / 32) + j
    const uint32_t j = x % (D / 32), ch = 32 * j + 8 * (x / (D / 32));
    const size_t   row = cache_row(c, page, head, 0);
    const uint8_t*  codes  = c.codes[0] + row * (D / 2) + x * 4;
    const uint32_t* scales = c.scales[0] + row * (D / G) + 32 * j / G;
    double          sum[8] = {};
    for(uint32_t b = r0; b < rows; b += kRows * kAhead) {
        uint32_t w[kAhead], s[kAhead];
#pragma unroll
        for(int i = 0; i < kAhead; ++i) {
            const uint32_t r = min(b + i * kRows, rows - 1);
            w[i] = *reinterpret_cast<const uint32_t*>(codes + (size_t)r * (D / 2));
            s[i] = scales[(size_t)r * (D / G)];
        }
#pragma unroll
        for(int i = 0; i < kAhead; ++i) {
            if(b + i * kRows >= rows) continue;
            const double step = half_bits_to_float(s[i] & 0xFFFFu);
            const double mid  = half_bits_to_float(s[i] >> 16);
#pragma unroll
            for(int e = 0; e < 8; ++e)
                sum[e] += fma(step, (double)((int)(w[i] >> (4 * e) & 15u) - 8), mid);
        }
    }
    int  e2 = kNoPower;
    bool ok = true;
#pragma unroll
    for(int e = 0; e < 8; ++e) {
        if constexpr(kLanes == 8) sum[e] = add_across<8>(sum[e]);
        sum[e] = add_across<32>(add_across<16>(sum[e])) / (double)rows;
        ok     = ok && fabs(sum[e]) < (double)INFINITY;
        e2     = max(e2, power_for(sum[e]));
    }
    ok = __ballot(!ok) == 0;
    e2 = wave_max_i32(e2); // (its rows' lanes all hold the same)
    const bool some = ok && e2 != kNoPower;
    if(r0 != 0) return;
    uint32_t q[2] = {0, 0};
    if(some)
#pragma unroll
        for(int e = 0; e < 8; ++e)
            q[e / 4] |= ((uint32_t)(int)rint(ldexp(sum[e], -e2)) & 0xFFu) << (8 * (e % 4));
    const size_t to = (size_t)page * c.kv_heads + head;
    *reinterpret_cast<v2i*>(a.codes + to * D + ch) = v2i{(int)q[0], (int)q[1]};
    if(lane == 0) a.scales[to] = !ok ? NAN : some ? ldexpf(1.f, e2) : 0.f;
}

// Values of page keys: 4 channels a thread.
__global__ void __launch_bounds__(kWaveThreads)
    kv4_page_keys_kernel(Kv4PageKeysArgs a, uint32_t count)
{
    const uint32_t i = blockIdx.x * kWaveThreads + threadIdx.x;
    if(i >= count) return;
    const uint32_t per  = a.kv_heads * (a.head_dim / 4);
    const int32_t  page = a.list[i / per];
    if(page < 0 || (uint32_t)page >= a.pages) return;
    const uint32_t at = i % per;
    const int32_t  w = *reinterpret_cast<const int32_t*>(
        a.codes + (size_t)page * a.kv_heads * a.head_dim + 4 * at);
    const float s = a.scales[(size_t)page * a.kv_heads + at / (a.head_dim / 4)];
    *reinterpret_cast<v4f*>(a.out + (size_t)i * 4)
        = v4f{(float)(int8_t)w * s, (float)(int8_t)(w >> 8) * s, (float)(int8_t)(w >> 16) * s,
              (float)(w >> 24) * s};
}

// ---------------------------------------------------------------------------
// The pages that suit a query: score = scale of the page key * (its codes . the query's
// codes), the query being the sum of the key head's query heads in 8 bits.  The dot
// product is a whole number below 2^21 and the scale a power of two, so a score is exact
// in fp32 and equal scores are equal everywhere.  A block takes one key head of a sequence:
// scores, lane = page, as whole numbers in their order; then the keep-th largest by its
// bytes, from counts of their values; then the columns in order.
//
// Up to kOneBlockPages columns the scores stay in LDS and one launch does it all; with more,
// or with more than half as many and few blocks, a launch before it computes the scores with a
// block for each 256 pages, since one block reads page keys at some 50 GB/s.  us in one launch
// and in two, heads of 128, 8 key heads: one sequence of 2048 pages 10.6, 11; of 4096 15.8,
// 11.6; 32 sequences of 4096 40, 45.
// ---------------------------------------------------------------------------
constexpr int      kSelectThreads = 1024;
constexpr uint32_t kOneBlockPages = 4096;

// The query's codes of one key head into LDS; all threads of the block.
template <int D>
__device__ __forceinline__ void query_codes(const Kv4SelectArgs& a, uint32_t seq, uint32_t head,
                                            int* powers, uint32_t* codes)
{
    constexpr int  kNotFinite = 5000;
    const uint32_t per        = a.heads / a.kv_heads;
    double         sum        = 0.0;
    if(threadIdx.x < D) {
        const uint16_t* q = a.q + (size_t)seq * a.ldq + (size_t)head * per * D + threadIdx.x;
#pragma unroll 8
        for(uint32_t h = 0; h < per; ++h) sum += (double)half_bits_to_float(q[(size_t)h * D]);
        const int e = wave_max_i32(fabs(sum) < (double)INFINITY ? power_for(sum) : kNotFinite);
        if(threadIdx.x % kWave == 0) powers[threadIdx.x / kWave] = e;
    }
    __syncthreads();
    if(threadIdx.x < D) {
        const int  e2   = D == 128 ? max(powers[0], powers[1]) : powers[0];
        const bool some = e2 != kNoPower && e2 != kNotFinite;
        reinterpret_cast<int8_t*>(codes)[threadIdx.x]
            = some ? (int8_t)(int)rint(ldexp(sum, -e2)) : 0;
    }
    __syncthreads();
}

// Scores of columns first .. end - 1 of `have`, as whole numbers in the scores' order, into
// `order`: D / 16 lanes a page, 16 bytes each, so that a wave reads whole lines (a lane a page
// takes 10 us for 2048 pages and not 4), THREADS lanes in all, 8 pages of each on their way (16
// gain nothing with 2048 pages and lose 2 us with few), the first ones while the query's codes
// are made (32 sequences of up to 1000 pages 10.6 us, 8.5 .. 10).
template <int D, int THREADS>
__device__ __forceinline__ void page_orders(const Kv4SelectArgs& a, uint32_t seq, uint32_t head,
                                            uint32_t first, uint32_t end, uint32_t have,
                                            int* powers, uint32_t* codes, uint32_t* order)
{
    constexpr uint32_t kLanes = D / 16, kGroups = THREADS / kLanes, kAhead = 8;
    const uint32_t     sub = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
    const int32_t*     from = a.table + (size_t)seq * a.table_ld;
    v4i                q{};
    for(uint32_t b0 = first; b0 < end; b0 += kGroups * kAhead) {
        const uint32_t c0 = b0 + group;
        int32_t        page[kAhead];
        v4i            k[kAhead];
        float          s[kAhead];
#pragma unroll
        for(uint32_t x = 0; x < kAhead; ++x) {
            const uint32_t c = c0 + x * kGroups;
            page[x]          = c < end ? from[c] : -1;
        }
#pragma unroll
        for(uint32_t x = 0; x < kAhead; ++x) {
            if(page[x] < 0 || (uint32_t)page[x] >= a.pages) page[x] = -1;
            const size_t at = (size_t)max(page[x], 0) * a.kv_heads + head;
            k[x]            = reinterpret_cast<const v4i*>(a.codes + at * D)[sub];
            s[x]            = a.scales[at];
        }
        if(b0 == first) {
            query_codes<D>(a, seq, head, powers, codes);
            q = reinterpret_cast<const v4i*>(codes)[sub];
        }
#pragma unroll
        for(uint32_t x = 0; x < kAhead; ++x) {
            int32_t dot = 0;
#pragma unroll
            for(int e = 0; e < 4; ++e) dot = __builtin_amdgcn_sdot4(k[x][e], q[e], dot, false);
            dot += dpp_mov_i32<kDppQuadXor1>(dot);
            dot += dpp_mov_i32<kDppQuadXor2>(dot);
            if constexpr(kLanes == 8) dot += dpp_mov_i32<kDppRowHalfMirror>(dot);
            float score = page[x] >= 0 ? (float)dot * s[x] + 0.f : -INFINITY; // no -0
            if(!(score == score)) score = -INFINITY;
            const uint32_t c = c0 + x * kGroups;
            if(c + 1 == have) score = INFINITY; // the last page is always taken
            const uint32_t u = __float_as_uint(score);
            if(sub == 0 && c < end) order[c] = (u >> 31) != 0 ? ~u : u | 0x80000000u;
        }
    }
}

template <int D>
__global__ void __launch_bounds__(kWaveThreads)
    kv4_score_kernel(Kv4SelectArgs a, uint32_t* __restrict__ order, uint32_t parts)
{
    __shared__ int     powers[2];
    __shared__ alignas(16) uint32_t codes[D / 4];
    const uint32_t unit = blockIdx.x / parts, part = blockIdx.x % parts; // (sequence, key head)
    const uint32_t seq = unit / a.kv_heads, head = unit % a.kv_heads;
    const uint32_t len  = clamped(a.lens[seq], a.table_cols << a.page_shift);
    const uint32_t have = (len + (1u << a.page_shift) - 1) >> a.page_shift;
    if(have <= a.keep || part * kWaveThreads >= have) return; // all of them, or none here
    const uint32_t first = part * kWaveThreads;
    page_orders<D, kWaveThreads>(a, seq, head, first, min(first + kWaveThreads, have), have,
                                 powers, codes, order + (size_t)unit * a.table_cols);
}

// SCORED: `order` holds the scores.
template <int D, bool SCORED>
__global__ void __launch_bounds__(kSelectThreads)
    kv4_select_kernel(Kv4SelectArgs a, const uint32_t* __restrict__ order)
{
    constexpr int       kWaves = kSelectThreads / kWave;
    __shared__ uint32_t scores[SCORED ? 1 : kOneBlockPages];
    __shared__ int      powers[2];
    __shared__ alignas(16) uint32_t codes[D / 4];
    __shared__ uint32_t count[256], part[kWaves], bin, above, same;
    const int           lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const uint32_t      unit = blockIdx.x, seq = unit / a.kv_heads, head = unit % a.kv_heads;
    const uint32_t      len  = clamped(a.lens[seq], a.table_cols << a.page_shift);
    const uint32_t      have = (len + (1u << a.page_shift) - 1) >> a.page_shift;
    const int32_t*      from = a.table + (size_t)seq * a.table_ld;
    int32_t*            to   = a.chosen + (size_t)unit * a.keep;
    if(head == 0 && threadIdx.x == 0)
        a.lens_out[seq]
            = (int32_t)(have > a.keep ? len - ((have - a.keep) << a.page_shift) : len);
    if(have <= a.keep) {
        for(uint32_t i = threadIdx.x; i < a.keep; i += kSelectThreads)
            to[i] = i < have ? from[i] : -1;
        return;
    }
    if constexpr(!SCORED)
        page_orders<D, kSelectThreads>(a, seq, head, 0, have, have, powers, codes, scores);
    const uint32_t* mine = SCORED ? order + (size_t)unit * a.table_cols : scores;
    // ---- the keep-th largest, byte by byte from the top -------------------------------
    uint32_t        least = 0, mask = 0, left = a.keep; // of those that begin like `least`
    for(int shift = 24; shift >= 0; shift -= 8) {
        for(uint32_t i = threadIdx.x; i < 256; i += kSelectThreads) count[i] = 0;
        __syncthreads();
        for(uint32_t i = threadIdx.x; i < have; i += kSelectThreads) {
            const uint32_t u = mine[i];
            if((u & mask) == least) atomicAdd(&count[u >> shift & 255u], 1u);
        }
        __syncthreads();
        if(wave == 0) { // lane: bins 255 - 4 lane and the three below
            uint32_t n[4], sum = 0;
#pragma unroll
            for(int e = 0; e < 4; ++e) sum += n[e] = count[255 - 4 * lane - e];
            const uint32_t s      = lanes_sum(sum);
            uint32_t       before = s - sum;
            if(before < left && s >= left) { // one lane
#pragma unroll
                for(int e = 0; e < 4; ++e) {
                    if(before < left && before + n[e] >= left) {
                        bin   = 255 - 4 * lane - e;
                        above = before;
                        same  = n[e];
                    }
                    before += n[e];
                }
            }
        }
        __syncthreads();
        least |= bin << shift;
        mask |= 255u << shift;
        left -= above;
        if(same == left) break; // all that begin like it
    }
    // ---- the columns above it, and the first `left` of those that begin like it ---------
    constexpr uint32_t kEach = 4; // columns a thread, one after the other
    uint32_t           equal = 0, out = 0; // up to here
    for(uint32_t i0 = 0; i0 < have; i0 += kSelectThreads * kEach) {
        const uint32_t i = i0 + threadIdx.x * kEach;
        uint32_t       u[kEach], eq = 0, gt = 0;
#pragma unroll
        for(uint32_t x = 0; x < kEach; ++x) {
            u[x] = i + x < have ? mine[i + x] & mask : 0;
            eq += i + x < have && u[x] == least ? 1u : 0u;
            gt += u[x] > least ? 1u : 0u;
        }
        const uint32_t own = gt << 16 | eq, s = lanes_sum(own); // at most 4096 of each
        __syncthreads();
        if(lane == kWave - 1) part[wave] = s;
        __syncthreads();
        uint32_t before = s - own, all = 0;
#pragma unroll
        for(int w = 0; w < kWaves; ++w) {
            if(w < wave) before += part[w];
            all += part[w];
        }
        uint32_t e = equal + (before & 0xFFFFu); // equals before the column
        // places: what is above, and the equals so far up to `left`
        uint32_t place = out + (before >> 16) + min(e, left) - min(equal, left);
#pragma unroll
        for(uint32_t x = 0; x < kEach; ++x) {
            const bool is = i + x < have && u[x] == least;
            if(u[x] > least || (is && e < left)) to[place++] = from[i + x];
            e += is ? 1u : 0u;
        }
        out += (all >> 16) + min(equal + (all & 0xFFFFu), left) - min(equal, left);
        equal += all & 0xFFFFu;
    }
}

// Blocks for so many tokens to place, or columns whose pages may come back: one for few, since
// each finds the running sums by itself.
uint32_t blocks_for(uint64_t items)
{
    if(items <= 8 * kSeqs) return 1;
    return (uint32_t)std::min<uint64_t>(256, (items + kSeqs - 1) / kSeqs);
}

} // namespace

hipError_t launch_kv4_extend(const Kv4ExtendArgs& a, hipStream_t stream)
{
    const uint32_t blocks = blocks_for(a.tokens);
    if(blocks == 1 || (a.lens_out != a.lens && a.count_out != a.count)) {
        kv4_extend_kernel<true, true><<<blocks, kSeqs, 0, stream>>>(a);
        return hipGetLastError();
    }
    kv4_extend_kernel<true, false><<<blocks, kSeqs, 0, stream>>>(a);
    kv4_extend_kernel<false, true><<<1, kSeqs, 0, stream>>>(a);
    return hipGetLastError();
}

hipError_t launch_kv4_trim(const Kv4TrimArgs& a, hipStream_t stream)
{
    const uint32_t blocks = blocks_for((uint64_t)a.seqs * a.table_cols);
    if(blocks == 1 || (a.lens_out != a.lens && a.lens_out != a.keep && a.count_out != a.count)) {
        kv4_trim_kernel<true, true><<<blocks, kSeqs, 0, stream>>>(a);
        return hipGetLastError();
    }
    kv4_trim_kernel<true, false><<<blocks, kSeqs, 0, stream>>>(a);
    kv4_trim_kernel<false, true><<<1, kSeqs, 0, stream>>>(a);
    return hipGetLastError();
}

hipError_t launch_kv4_summarize(const w8a8_kv4_cache& c, const Kv4SummarizeArgs& a,
                                hipStream_t stream)
{
    const uint64_t pages = kv4_touched_pages(a.tokens, a.seqs, c.page_size);
    const uint32_t waves = kWaveThreads / kWave;
    const uint32_t blocks = (uint32_t)((pages * c.kv_heads + waves - 1) / waves);
    with_widths(c, [&](auto d, auto g) {
        kv4_summarize_kernel<d(), g()><<<blocks, kWaveThreads, 0, stream>>>(view(c), a, c.pages);
    });
    return hipGetLastError();
}

hipError_t launch_kv4_page_keys(const Kv4PageKeysArgs& a, hipStream_t stream)
{
    const uint32_t count = a.count * a.kv_heads * (a.head_dim / 4);
    kv4_page_keys_kernel<<<(count + kWaveThreads - 1) / kWaveThreads, kWaveThreads, 0, stream>>>(
        a, count);
    return hipGetLastError();
}

size_t kv4_select_workspace_bytes(uint32_t seqs, uint32_t kv_heads, uint32_t cols, uint32_t keep)
{
    const uint64_t units = (uint64_t)seqs * kv_heads;
    if(cols <= keep || cols <= kOneBlockPages / 2 || (cols <= kOneBlockPages && units >= 128))
        return 0; // one launch
    return units * cols * 4;
}

hipError_t launch_kv4_select(const Kv4SelectArgs& a, hipStream_t stream)
{
    const uint32_t units = a.seqs * a.kv_heads;
    auto*          order = static_cast<uint32_t*>(a.ws);
    const auto     run   = [&](auto d) {
        if(kv4_select_workspace_bytes(a.seqs, a.kv_heads, a.table_cols, a.keep) != 0) {
            const uint32_t parts = (a.table_cols + kWaveThreads - 1) / kWaveThreads;
            kv4_score_kernel<d()><<<units * parts, kWaveThreads, 0, stream>>>(a, order, parts);
            kv4_select_kernel<d(), true><<<units, kSelectThreads, 0, stream>>>(a, order);
        } else
            kv4_select_kernel<d(), false><<<units, kSelectThreads, 0, stream>>>(a, order);
    };
    if(a.head_dim == 64)
        run(std::integral_constant<int, 64>());
    else
        run(std::integral_constant<int, 128>());
    return hipGetLastError();
}

} // namespace w8a8
