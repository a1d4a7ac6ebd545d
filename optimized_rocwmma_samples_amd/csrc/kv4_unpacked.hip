// kv4_unpacked.hip -- attention of long chunks over the paged 4-bit cache, for gfx950: their
// sequences' keys and values are unpacked to fp16 once, and the tiles of attention.hip run
// over them.
//
// Unpacking costs 4 bytes written and read again for each of the cache's, some 4 % of the time
// of a chunk of 2048 tokens with four query heads a key head; unpacked by each block where it is
// used it would be a fifth of every block's instructions.
//
// The work of a sequence is cut into units of 128 rows of one query head over their key
// tiles.  The blocks of one gang, the query heads of a key head (and neighbouring tiles of
// rows, where those are fewer than four), take the same keys at the same time, so that all but
// the first find them in their XCD's L2.  All gangs' key tiles lie in one line, which is cut
// into equal runs, one a gang of blocks, all resident: any mix of chunks keeps the chip evenly
// busy.  What a cut leaves of a unit is joined by another launch.
//
// MI355X, 2048 new of 18432 tokens, 32/8 heads of 128: unpacking 22 us (75 MB written at 3 TB/s
// beside 17 read), attention 605 to 710 by the card's clock (584 GFLOP, 820 to 960 TFLOP/s, of
// the 1390 of a large product; matrix instructions fill 49 % of the cycles and vector
// instructions 49 %, waves wait for 35 % of their time), joining 20 (up to 100 MB of partials).  By the kernel of few rows, which
// unpacks for every 64 rows anew, the same chunk took 1190.
#include "attention_tile.hpp"
#include "kv4_chunks.hpp"

#include <algorithm>

namespace w8a8 {
namespace {

constexpr uint64_t kMostBytes = 1ull << 30;   // of unpacked keys and values

template <int D>
constexpr int kKeysOf = 4096 / D;

// ---- which sequences ------------------------------------------------------------------
struct Which {
    uint32_t count, rows; // sequences that are unpacked, and their rows in all
};

// Finds them, one wave: emit(sequence, is one, place in the list, entry), lane = sequence.
template <class E>
__device__ __forceinline__ Which find_longs(const ChunkArgs& a, const LongList& l, E emit)
{
    const uint32_t lane = threadIdx.x % kWave;
    Which          w{};
    bool           full = false;
    for(uint32_t i0 = 0; i0 < a.seqs; i0 += kWave) {
        const uint32_t i = i0 + lane;
        Chunk          c{};
        if(i < a.seqs) c = chunk_of(a, i, l.most_len);
        const bool     want = (uint64_t)c.fresh * l.per > kFewRows && c.len >= c.fresh;
        const uint32_t pad  = (l.keys - (c.len - c.fresh) % l.keys) % l.keys;
        // (one row more than there is room for is as good as any number)
        const uint32_t need
            = want ? min((c.len + pad + l.keys - 1) / l.keys * l.keys, l.rows + 1) : 0;
        const uint32_t s  = lanes_sum(need);
        bool           ok = want && !full && s <= l.rows - w.rows;
        const uint64_t in = __ballot(ok);
        const uint32_t at = w.count + __builtin_popcountll(in & ((1ull << lane) - 1));
        ok                = ok && at < l.most; // more only where starts do not ascend
        if(i < a.seqs) emit(i, ok, at, Long{i, w.rows + s - need, need, pad, c, 0});
        const uint64_t oks = __ballot(ok);
        full               = full || oks != __ballot(want); // those behind it find no room
        w.count += __builtin_popcountll(oks);
        if(oks != 0) w.rows += __builtin_amdgcn_readlane((int)s, 63 - __builtin_clzll(oks));
    }
    return w;
}

// The list of many sequences; of up to 64 the next kernel's blocks find them by themselves,
// which saves 5 us.
__global__ void __launch_bounds__(kWave) kv4_long_kernel(ChunkArgs a, LongList l)
{
    const Which w = find_longs(a, l, [&](uint32_t i, bool ok, uint32_t at, const Long& x) {
        if(ok) l.list[at] = x;
        l.flags[i] = ok;
    });
    if(threadIdx.x == 0) *reinterpret_cast<Which*>(l.total) = w;
}

// ---- unpacking ------------------------------------------------------------------------
struct Unpacked {
    uint16_t *k, *v;
    uint32_t* missing; // bit i of word j: row 32 j + i has no token
};

// 8 values of a dword of codes, what kv4_load gives, but NaN where the scale or the offset is
// an infinity (whose product with 0 is NaN; added to the offset it reaches all codes).
__device__ __forceinline__ v4i unpacked(uint32_t w, uint32_t pair)
{
    const float s = half_bits_to_float(pair & 0xFFFFu);
    const float o = half_bits_to_float(pair >> 16), mid = fmaf(o, 0.f, fmaf(s, 0.f, o));
    v4i         out;
#pragma unroll
    for(int j = 0; j < 4; ++j)
        out[j] = (int)finite_halves(fmaf(s, (float)(w >> (8 * j) & 15u) - 8.f, mid),
                                    fmaf(s, (float)(w >> (8 * j + 4) & 15u) - 8.f, mid));
    return out;
}

// A block takes 32 rows of one key head at a time; a thread 8 channels of a row's keys and
// values.  The unpacked rows of a sequence's key head lie together.
template <int D, int G>
__global__ void __launch_bounds__(256)
    kv4_unpack_kernel(CacheView c, ChunkArgs a, LongList l, Unpacked u, uint32_t pages)
{
    constexpr uint32_t kPer = D / 8, kRound = 256 / kPer; // chunks of a row, rows a round
    __shared__ Long    longs[kWave];
    __shared__ Which   found;
    const uint32_t     lane = threadIdx.x % kWave;
    const bool         here = a.seqs <= kWave; // the list is made here
    if(here) {
        if(threadIdx.x < kWave) {
            const bool  first = blockIdx.x == 0;
            const Which w = find_longs(a, l, [&](uint32_t i, bool ok, uint32_t at, const Long& x) {
                if(ok) longs[at] = x;
                if(ok && first) l.list[at] = x;
                if(first) l.flags[i] = ok;
            });
            if(lane == 0) {
                found = w;
                if(first) *reinterpret_cast<Which*>(l.total) = w;
            }
        }
        __syncthreads();
    }
    const Which     w    = here ? found : *reinterpret_cast<const Which*>(l.total);
    const Long*     list = here ? longs : l.list;
    const uint32_t  count = w.count, work = w.rows / 32 * c.kv_heads;
    for(uint32_t at = blockIdx.x; at < work; at += gridDim.x) {
        const uint32_t row0 = at / c.kv_heads * 32, head = at % c.kv_heads;
        uint32_t       which = 0; // the last sequence that begins at or before row0
        for(uint32_t i0 = 0; i0 < count; i0 += kWave) {
            const uint64_t in
                = __ballot(i0 + lane < count && list[min(i0 + lane, count - 1)].base <= row0);
            which += __builtin_popcountll(in);
        }
        const Long&    x = list[which - 1];
        const uint32_t from = row0 - x.base; // of the sequence's rows
        auto           page_of = [&](uint32_t r) { // of the token in row r, or -1
            const uint32_t t = from + r - x.pad;
            if(from + r < x.pad || t >= x.c.len) return -1;
            const int32_t p = a.table[(size_t)x.seq * a.table_ld + (t >> c.page_shift)];
            return p >= 0 && (uint32_t)p < pages ? p : -1;
        };
        if(head == 0 && threadIdx.x < kWave) {
            const uint64_t gone = __ballot(lane < 32 && page_of(lane % 32) < 0);
            if(lane == 0) u.missing[row0 / 32] = (uint32_t)gone;
        }
        const size_t to0 = (size_t)x.base * c.kv_heads * D + ((size_t)head * x.need + from) * D;
        const uint32_t chunk = threadIdx.x % kPer;
#pragma unroll
        for(uint32_t r0 = 0; r0 < 32; r0 += kRound) {
            const uint32_t r = r0 + threadIdx.x / kPer;
            const int32_t  page = page_of(r);
            v4i            k = {}, v = {};
            if(page >= 0) {
                const size_t row
                    = cache_row(c, page, head, (from + r - x.pad) & (c.page_size - 1));
                // dword of channels 8 chunk ..: of keys (chunk % 4, chunk / 4) of [4][D / 32]
                const size_t kb = row * (D / 2) + chunk % 4 * (D / 8) + chunk / 4 * 4;
                k = unpacked(*reinterpret_cast<const uint32_t*>(c.codes[0] + kb),
                             c.scales[0][row * (D / G) + chunk * 8 / G]);
                v = unpacked(
                    *reinterpret_cast<const uint32_t*>(c.codes[1] + row * (D / 2) + chunk * 4),
                    c.scales[1][row * (D / G) + chunk * 8 / G]);
            }
            const size_t to = to0 + (size_t)r * D + chunk * 8;
            *reinterpret_cast<v4i*>(u.k + to) = k;
            *reinterpret_cast<v4i*>(u.v + to) = v;
        }
    }
}

// ---- attention ------------------------------------------------------------------------
struct Gang {
    uint32_t members, heads, tiles; // blocks of a gang: query heads x tiles of rows
};

template <int D>
__global__ void __launch_bounds__(kThreads, 3)
    attention_unpacked_kernel(ChunkArgs a, LongList l, Unpacked u, Runs runs, Gang gang,
                              uint32_t kv_heads)
{
    constexpr uint32_t kKeys = kKeysOf<D>;
    constexpr int      kBlocks = D / 32;
    __shared__ alignas(256) uint8_t lds[2 * 2 * kKeys * D * 2];
    const uint32_t lane = threadIdx.x % kWave;
    // blocks go round the 8 XCDs: an XCD has whole gangs, and neighbouring runs
    const uint32_t run    = blockIdx.x % 8 * (runs.count / 8) + blockIdx.x / 8 / gang.members;
    const uint32_t member = blockIdx.x / 8 % gang.members;
    const uint32_t count  = l.total[0], per = a.heads / kv_heads;
    const uint32_t groups = kv_heads * (per / gang.heads), rows = gang.tiles * kRows;

    // A sequence's row tiles of a gang see more and more keys, the last one all of them.
    auto tiles_of = [&](const Long& x) { return (x.c.fresh + rows - 1) / rows; };
    auto keys_of  = [&](const Long& x, uint32_t tile) { // key tiles
        const uint32_t end = min((tile + 1) * rows, x.c.fresh); // of its rows
        return (x.c.len - x.c.fresh + x.pad + end + kKeys - 1) / kKeys;
    };
    auto all_keys = [&](const Long& x) { // of all its row tiles
        const uint32_t n = tiles_of(x), before = (x.c.len - x.c.fresh + x.pad) / kKeys;
        return (n - 1) * before + rows / kKeys * ((n - 1) * n / 2) + keys_of(x, n - 1);
    };

    // ---- the gang's run ----------------------------------------------------------------
    auto scan = [&](uint32_t i0, uint32_t& n, uint32_t& s) { // 64 sequences' key tiles
        n = i0 + lane < count ? all_keys(l.list[i0 + lane]) * groups : 0;
        s = lanes_sum(n);
        return (uint32_t)__builtin_amdgcn_readlane(s, kWave - 1);
    };
    uint32_t n, s, all = 0;
    for(uint32_t i = 0; i < count; i += kWave) all += scan(i, n, s);
    const uint32_t q = all / runs.count, r = all % runs.count;
    uint32_t       at = run * q + min(run, r), left = q + (run < r ? 1 : 0);
    uint32_t*      tasks = runs.tasks + (size_t)run * gang.members + member;
    uint32_t       mine  = 0; // the join's tasks with what this block's run cuts
    if(left == 0) {
        if(threadIdx.x == 0) *tasks = 0;
        return;
    }
    const uint32_t end = at + left;
    uint32_t       which = 0;
    for(uint32_t i = 0; i < count; i += kWave) {
        const uint32_t sum = scan(i, n, s);
        if(at < sum) {
            const int f = __builtin_ctzll(__ballot(s > at));
            at -= __builtin_amdgcn_readlane(s, f) - __builtin_amdgcn_readlane(n, f);
            which = i + f;
            break;
        }
        at -= sum;
    }
    Long     x     = l.list[which];
    uint32_t group = at / all_keys(x), tile = 0;
    at             = at % all_keys(x);
    while(at >= keys_of(x, tile)) at -= keys_of(x, tile++);

    const float c = a.scale * 1.44269504088896341f;
    while(left != 0) {
        const uint32_t keys = keys_of(x, tile), take = min(left, keys - at);
        const uint32_t head0 = group * gang.heads, head = head0 + member % gang.heads;
        const uint32_t row0  = (tile * gang.tiles + member / gang.heads) * kRows;
        const bool     from_start = at == 0, ends = at + take == keys;
        if(row0 < x.c.fresh) {
            TileRows t;
            t.q     = a.q + (size_t)(x.c.begin + row0) * a.ldq + head * D;
            t.ldq   = a.ldq;
            t.ldk   = t.ldv = D;
            t.rows  = min((uint32_t)kRows, x.c.fresh - row0);
            t.first = x.c.len - x.c.fresh + x.pad + row0;
            t.keys  = x.c.len + x.pad;
            // along the line the last keys come first
            t.to   = min(keys - at, (t.first + t.rows + kKeys - 1) / kKeys);
            t.from = keys - at - take;
            const size_t kv
                = (size_t)x.base * kv_heads * D + (size_t)(head / per) * x.need * D;
            t.k = u.k + kv;
            t.v = u.v + kv;
            float m = -INFINITY, sum = 0.f, mc = 0.f;
            v16f  o[kBlocks] = {};
            if(t.to > t.from)
                attend<D, kKeys, true>(t, c, u.missing + x.base / 32, lds, m, sum, mc, o);
            const v2f sums = both_halves(sum);
            sum            = sums[0] + sums[1];
            const uint32_t half = lane / 32, row = threadIdx.x / kWave * 32 + lane % 32;
            if(row < t.rows) {
                if(ends && from_start) {
                    const float inv = sum != 0.f ? 1.f / sum : 0.f;
                    uint16_t*   out
                        = a.out + (size_t)(x.c.begin + row0 + row) * a.ldo + head * D + 4 * half;
#pragma unroll
                    for(int b = 0; b < kBlocks; ++b)
#pragma unroll
                        for(int i = 0; i < 16; i += 4)
                            *reinterpret_cast<v2i*>(out + 32 * b + 2 * i)
                                = v2i{(int)finite_halves(o[b][i] * inv, o[b][i + 1] * inv),
                                      (int)finite_halves(o[b][i + 2] * inv, o[b][i + 3] * inv)};
                } else {
                    const size_t slot
                        = ((size_t)(2 * run + (from_start ? 1 : 0)) * gang.members + member) * kRows
                          + row;
#pragma unroll
                    for(int b = 0; b < kBlocks; ++b)
#pragma unroll
                        for(int i = 0; i < 16; i += 4)
                            *reinterpret_cast<v4f*>(runs.o + slot * D + 32 * b + 2 * i + 4 * half)
                                = v4f{o[b][i], o[b][i + 1], o[b][i + 2], o[b][i + 3]};
                    if(half == 0) *reinterpret_cast<v2f*>(runs.ml + slot * 2) = v2f{m * c, sum};
                }
            }
        }
        left -= take;
        if(!ends && from_start && threadIdx.x == 0) { // goes on behind the run: up to which one
            const uint32_t last = end - 1 + (keys - at - take); // its last key tile
            const uint32_t to = last < r * (q + 1) ? last / (q + 1) : r + (last - r * (q + 1)) / q;
            if(member == 0) runs.cut[run] = {to + 1, x.c.begin, tile * rows, x.c.fresh, head0, {}};
            if(row0 < x.c.fresh)
                mine = join_tasks<D>(to + 1 - run, min((uint32_t)kRows, x.c.fresh - row0));
        }
        if(left == 0) break;
        at = 0;
        if(++tile == tiles_of(x)) {
            tile = 0;
            if(++group == groups) {
                group = 0;
                x     = l.list[++which];
            }
        }
        __syncthreads(); // all waves are done with the tiles in LDS
    }
    if(threadIdx.x == 0) *tasks = mine;
}

} // namespace

UnpackedLayout unpacked_layout(const w8a8_kv4_cache& c, uint32_t seqs, uint32_t tokens,
                               uint32_t heads, uint32_t table_cols, uint32_t max_new)
{
    UnpackedLayout u{};
    const uint32_t per = heads / c.kv_heads, d = c.head_dim, keys = 4096 / d;
    if((uint64_t)std::min(max_new, tokens) * per <= kFewRows) return u;
    // no more sequences than have that many new tokens, each of at most the table's columns
    const uint64_t longs = std::min<uint64_t>(seqs, tokens / (kFewRows / per + 1));
    const uint64_t each  = ((uint64_t)table_cols * c.page_size + 2 * keys - 1) / keys * keys;
    u.room               = (uint32_t)longs;
    const uint64_t cap   = kMostBytes / (4ull * c.kv_heads * d) / keys * keys;
    u.rows               = (uint32_t)std::min(longs * each, cap);
    if(u.rows == 0 || table_cols == 0) return UnpackedLayout{};
    // the gang: as many of a key head's query heads as divide them, and neighbouring tiles
    // of rows up to four blocks
    u.heads = 1;
    for(uint32_t h = 2; h <= 16; ++h)
        if(per % h == 0) u.heads = h;
    u.tiles   = u.heads >= 4 ? 1 : 4 / u.heads;
    u.members = u.heads * u.tiles;
    u.runs    = kUnpackedBlocks / 8 / u.members * 8;
    // the line of key tiles is counted in 32 bits, whatever the starts are (only some ten
    // thousand query heads on one key head could make it longer)
    if((tokens / (u.tiles * kRows) + 1ull) * (u.rows / keys) * c.kv_heads * (per / u.heads)
       > 0xFFFFFFFFull)
        return UnpackedLayout{};
    size_t at   = 0;
    auto   room = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    const size_t slots = (size_t)u.runs * 2 * u.members * kRows;
    u.o       = room(slots * d * 4);
    u.ml      = room(slots * 8);
    u.cut     = room(u.runs * sizeof(Piece));
    u.total   = room(8);
    u.list    = room(u.room * sizeof(Long));
    u.flags   = room(seqs);
    u.missing = room(u.rows / 32 * 4);
    u.k       = room((size_t)u.rows * c.kv_heads * d * 2);
    u.v       = room((size_t)u.rows * c.kv_heads * d * 2);
    u.bytes   = at;
    return u;
}

void launch_unpacked(const w8a8_kv4_cache& c, const ChunkArgs& a, const UnpackedLayout& u,
                     const Runs& runs, uint8_t* ws, hipStream_t stream)
{
    const LongList list{u.room, u.rows, reinterpret_cast<uint32_t*>(ws + u.total),
                        reinterpret_cast<Long*>(ws + u.list), ws + u.flags,
                        a.heads / c.kv_heads, a.table_cols * c.page_size,
                        4096 / c.head_dim};
    const Unpacked un{reinterpret_cast<uint16_t*>(ws + u.k), reinterpret_cast<uint16_t*>(ws + u.v),
                      reinterpret_cast<uint32_t*>(ws + u.missing)};
    const Gang     gang{u.members, u.heads, u.tiles};
    if(a.seqs > kWave) kv4_long_kernel<<<1, kWave, 0, stream>>>(a, list);
    const uint32_t groups = (uint32_t)std::min<uint64_t>((uint64_t)u.rows / 32 * c.kv_heads, 4096);
    with_widths(c, [&](auto d, auto g) {
        kv4_unpack_kernel<d(), g()><<<groups, 256, 0, stream>>>(view(c), a, list, un, c.pages);
    });
    const auto kernel
        = c.head_dim == 64 ? attention_unpacked_kernel<64> : attention_unpacked_kernel<128>;
    kernel<<<u.runs * u.members, kThreads, 0, stream>>>(a, list, un, runs, gang, c.kv_heads);
}

} // namespace w8a8
