// kv4_chunks.hpp -- what the two kernels of attention of chunks over the 4-bit cache share: the
// sequences of a call, which of them go which way, and the pieces that runs cut units into.
#pragma once

#include "kv4_device.hpp"

namespace w8a8 {
namespace {

// A sequence with more rows (new tokens x query heads a key head) than this has its keys and
// values unpacked to fp16 first, once, and then takes the prompts' tiles over them; the others
// unpack codes where they use them, each 64 rows again.  us, one sequence of 8192 tokens, 32/8
// heads of 128, unpacked where used and unpacked first: 260 rows (65 tokens) 47 .. 59 and
// 69 .. 73, 512 rows 50 .. 64 and 82 .. 88; 1024 rows take 90 unpacked first, twice the 512 rows'
// work where used.
constexpr uint32_t kFewRows = 512;

// One sequence of the call.
struct Chunk {
    uint32_t begin, fresh, len; // first row of q, new tokens, tokens in all
};

__device__ __forceinline__ Chunk chunk_of(const ChunkArgs& a, uint32_t i, uint32_t most)
{
    const int32_t b = min(max(a.starts[i], 0), (int32_t)a.tokens);
    const int32_t e = min(max(a.starts[i + 1], 0), (int32_t)a.tokens);
    return {(uint32_t)b, (uint32_t)max(e - b, 0), (uint32_t)max(min(a.lens[i], (int32_t)most), 0)};
}

// A sequence that is unpacked: its tokens are rows base + pad .. of the unpacked keys and
// values (`need` rows in all, whole key tiles), so that its first new token begins a tile.
struct Long {
    uint32_t seq, base, need, pad;
    Chunk    c;
    uint32_t unused; // 32 bytes, which no line of memory cuts
};

// Which sequences are unpacked; in the workspace.
struct LongList {
    uint32_t  most;  // the list's room
    uint32_t  rows;  // room for unpacked tokens
    uint32_t* total; // [0] sequences in the list, [1] their rows
    Long*     list;
    uint8_t*  flags; // [seqs] 1: in the list
    uint32_t  per, most_len, keys; // query heads a key head, tokens at the most, keys of a tile
};

} // namespace

// What the join needs of a unit that goes on behind the run it begins in: written, and read,
// where the run's tasks are not 0.
struct Piece {
    uint32_t last;  // run that has its last step, plus 1
    uint32_t token; // first row of q of its sequence
    uint32_t row0, rows; // its rows row0 .. of the sequence's `rows`
    uint32_t head;       // first query head
    uint32_t unused[3]; // 32 bytes, as above
};

// Whether the rows of a unit are joined by a block each, which takes all partials at a time, or
// 32 (64) by a block, which takes two after two.  One token of 2048 (16 partials of 4 rows):
// 6 us and 12; a batch of chunks whose units of 128 rows have 3 to 8 partials: 73 and 15.
__device__ __forceinline__ bool join_many(uint32_t partials, uint32_t rows)
{
    return partials > 16 || (partials > 8 && rows <= 64);
}
template <int D>
constexpr uint32_t kJoinRows = 2 * 256 / (D / 8);

template <int D>
__device__ __forceinline__ uint32_t join_tasks(uint32_t partials, uint32_t rows)
{
    return join_many(partials, rows) ? rows : (rows + kJoinRows<D> - 1) / kJoinRows<D>;
}

// Partials: slot 2 r of run r holds a unit that began before it, 2 r + 1 one that begins in it
// and goes on: fp32 [rows, head_dim], then (maximum, sum) of each row.
struct Runs {
    uint32_t count;
    float*   o;
    float*   ml;
    Piece*   cut;
    uint32_t* tasks; // the join's with each run's (and block's of it) cut unit
};

// The kernels over unpacked keys and values (kv4_unpacked.hip).
constexpr uint32_t kUnpackedBlocks = 3 * 256; // all resident: 3 a CU
struct UnpackedLayout {
    uint32_t runs, members, heads, tiles; // members = heads x tiles blocks share a run's keys
    uint32_t room, rows;                  // of the list, of unpacked tokens; 0: none
    size_t   o, ml, cut, total, list, flags, missing, k, v, bytes; // offsets
};
UnpackedLayout unpacked_layout(const w8a8_kv4_cache& c, uint32_t seqs, uint32_t tokens,
                               uint32_t heads, uint32_t table_cols, uint32_t max_new);
inline Runs unpacked_runs(const UnpackedLayout& u, uint8_t* ws, uint32_t* tasks)
{
    return {u.runs, reinterpret_cast<float*>(ws + u.o), reinterpret_cast<float*>(ws + u.ml),
            reinterpret_cast<Piece*>(ws + u.cut), tasks};
}
void launch_unpacked(const w8a8_kv4_cache& c, const ChunkArgs& a, const UnpackedLayout& u,
                     const Runs& runs, uint8_t* ws, hipStream_t stream);

} // namespace w8a8
