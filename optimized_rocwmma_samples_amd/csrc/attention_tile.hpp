// attention_tile.hpp -- the work of one block of attention: 128 query rows of one head, 32 a
// wave, over key tiles in LDS.  Used for whole prompts and for chunks of prompts whose cached
// keys and values were unpacked before; the mathematics and what bounds it stand in
// attention.hip.
#pragma once

#include "matrix_f16.hpp"
#include "w8a8_internal.hpp"

namespace w8a8 {
namespace {

typedef __attribute__((address_space(3))) v8h    lds_v8h_t;
typedef __attribute__((address_space(4))) uint32_t constant_u32_t;

constexpr int kBufferFlags = 0x00020000; // raw buffer, 32-bit data format
constexpr int kRows        = 128;        // query rows a block
constexpr int kWaves       = kRows / 32;
constexpr int kThreads     = kWaves * kWave;
constexpr uint32_t kCus    = 256;

// Blocks a CU.  Keys a tile are 4096 / D, whose scores leave registers for 3 waves a SIMD
// and more, or twice as many, two independent chains a wave, for 2.
template <int D, int KEYS>
constexpr int kBlocksOf = D * KEYS == 4096 ? 3 : 2;

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

// What a block works on: its rows, and the keys and values of its head, row by row.
struct TileRows {
    const uint16_t *q, *k, *v;
    uint32_t        ldq, ldk, ldv;
    uint32_t        rows;     // query rows, at most kRows
    uint32_t        first;    // position of the first of them: row i sees keys 0 .. first + i
    uint32_t        keys;     // keys there are
    uint32_t        from, to; // key tiles to take, the last one first
};

// One pass over the tiles: on return the wave's lane has its row's maximum m (mc = m c, 0
// while no score is finite), its own half of the sum l of probabilities and, of 32
// channels a block, the sum of their products with the values.  Where `first` is a multiple
// of KEYS each wave meets its diagonal in its first tile.  MASKED: a chunk's rows; bit i of
// missing[j] says that there is no key 32 j + i (whose values are zeros).
template <int D, int KEYS, bool MASKED>
__device__ __forceinline__ void attend(const TileRows& t, float c, const uint32_t* missing,
                                       uint8_t* lds, float& m, float& l, float& mc,
                                       v16f (&o)[D / 32])
{
    constexpr int kKeys      = KEYS;
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
    const uint32_t first = t.first + wave * 32; // position of the wave's first row
    const uint32_t qi    = first + col;         // and of the lane's

    // ---- tiles into LDS -------------------------------------------------------
    const uint32_t  ldkb = t.ldk * 2, ldvb = t.ldv * 2;
    uint32_t        ko[kLoads], vo[kLoads];
#pragma unroll
    for(int i = 0; i < kLoads; ++i) {
        const uint32_t tok = (wave * kLoads + i) * kRowsLoad + lane / kChunks;
        ko[i]              = tok * ldkb + key_chunk<D>(tok, lane % kChunks) * 16;
        vo[i]              = tok * ldvb + value_chunk<D>(tok, lane % kChunks) * 16;
    }
    const uint32_t lds0 = (uint32_t)(uintptr_t)lds;
    auto           issue = [&](int stage, uint32_t kt) {
        const uint32_t n = min((uint32_t)kKeys, t.keys - kt * kKeys);
        const v4i      rk = buffer(t.k + (size_t)kt * kKeys * t.ldk, (n - 1) * ldkb + D * 2);
        const v4i      rv = buffer(t.v + (size_t)kt * kKeys * t.ldv, (n - 1) * ldvb + D * 2);
        const uint32_t to = lds0 + stage * 2 * kTileBytes + wave * kLoads * 1024;
#pragma unroll
        for(int i = 0; i < kLoads; i += 2) load_lds(rk, to + i * 1024, ko[i], ko[i + 1]);
#pragma unroll
        for(int i = 0; i < kLoads; i += 2)
            load_lds(rv, to + kTileBytes + i * 1024, vo[i], vo[i + 1]);
    };

    issue(0, t.to - 1);

    // ---- the wave's query rows: lane = row, 8 channels from 16 step + 8 half ----
    // Zeros behind the last row.  Rows of a chunk may lie any distance apart; those of a prompt
    // no more than 2^24 values, which a buffer's 32-bit offsets hold.  The same us: chunks (2048
    // of 18432 tokens) 643 by addresses and 648 by a buffer, prompts (8192) 547 and 544.
    v8h            qf[kSteps] = {};
    const uint32_t qrow       = wave * 32 + col;
    if constexpr(MASKED) {
        const uint16_t* from = t.q + (size_t)qrow * t.ldq + half * 8;
        if(qrow < t.rows)
#pragma unroll
            for(int s = 0; s < kSteps; ++s)
                qf[s] = infinite_to_nan(*reinterpret_cast<const v8h*>(from + s * 16));
    } else {
        const __amdgpu_buffer_rsrc_t rq = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint16_t*>(t.q), 0, (int)((t.rows - 1) * t.ldq * 2 + D * 2), kBufferFlags);
#pragma unroll
        for(int s = 0; s < kSteps; ++s)
            qf[s] = __builtin_bit_cast(v8h, __builtin_amdgcn_raw_buffer_load_b128(
                                                rq, qrow * t.ldq * 2 + s * 32 + half * 16, 0, 0));
    }

    // LDS places of the lane's reads, in stage 0: of a key's first step and a value's first
    // block.  Rows are D * 2 bytes and LDS starts on such a border, so the swizzle of a
    // later step or block is one XOR away; all else are fixed distances.
    const uint32_t kat = lds0 + col * D * 2 + key_chunk<D>(col, half) * 16;
    const uint32_t tok0 = 4 * half + lane % 16 / 4, ch0 = lane / 16 % 2 * 16 + lane % 4 * 4;
    const uint32_t vat
        = lds0 + kTileBytes + tok0 * D * 2 + value_chunk<D>(tok0, ch0 / 8) * 16 + ch0 % 8 * 2;

    const uint64_t gaps_at = (uint64_t)missing; // uniform as well
    const auto*    gaps    = (const constant_u32_t*)(
        (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(gaps_at >> 32)) << 32
        | (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)gaps_at));
    for(uint32_t kt = t.to, stage = 0; kt-- > t.from; stage ^= 1) {
        // (a scalar load: a vector one would be waited for along with the next tile)
        uint32_t none[kSubs] = {};
        if constexpr(MASKED)
#pragma unroll
            for(int sub = 0; sub < kSubs; ++sub)
                none[sub] = gaps[__builtin_amdgcn_readfirstlane(kt * kSubs + sub)];
        wait_vmcnt<0>();   // this wave's part of the tile is there,
        wait_lgkmcnt0();   // and its reads of the tile before are done:
        __syncthreads();   // so are every wave's
        if(kt > t.from) issue(stage ^ 1, kt - 1);
        if(kt * kKeys > first + 31) continue; // all of the tile is later than the wave's rows

        const uint32_t off  = stage * 2 * kTileBytes;
        const bool     diag = (kt + 1) * kKeys > first; // some of it is later than some rows
        v16f           s[kSubs] = {};
        // Four key fragments on their way, in this order: left alone the compiler reads each into
        // the same registers and waits for it (8192 tokens 556 us for 545; two ahead 559, where
        // four are 554; six spill in the kernel over unpacked keys: 668 us, 676).
        constexpr int  kAhead = 4, kProducts = kSteps * kSubs;
        auto           key    = [&](int i) {
            return *(const lds_v8h_t*)(uintptr_t)(((kat + off) ^ (i / kSubs * 32))
                                                  + i % kSubs * 32 * D * 2);
        };
        v8h kf[kAhead];
#pragma unroll
        for(int i = 0; i < kAhead; ++i) kf[i] = key(i);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for(int i = 0; i < kProducts; ++i) {
            s[i % kSubs] = mfma(kf[i % kAhead], qf[i / kSubs], s[i % kSubs]);
            if(i + kAhead < kProducts) kf[i % kAhead] = key(i + kAhead);
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr(MASKED) {
#pragma unroll
            for(int sub = 0; sub < kSubs; ++sub) {
                if(none[sub] == 0) continue;
                const uint32_t gone = none[sub] >> (4 * half);
#pragma unroll
                for(int i = 0; i < 16; ++i)
                    if((gone >> (8 * (i / 4) + i % 4) & 1u) != 0) s[sub][i] = -INFINITY;
            }
        }
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
}

// The wave's rows written out: sums over the probabilities' sum, rounded to fp16.
template <int N>
__device__ __forceinline__ void write_rows(uint32_t rows, uint32_t row, float l, v16f (&o)[N],
                                           uint16_t* out)
{
    const int   half = threadIdx.x % kWave / 32;
    const v2f   ls  = both_halves(l);
    // The rounded probabilities may add up to a little more than l (2^-11 of it at the most),
    // which must not carry a mean of values of 65504 past fp16.
    const float inv = finite_halves_from_here(1.f / (ls[0] + ls[1]), o);
    if(row >= rows) return;
#pragma unroll
    for(int b = 0; b < N; ++b)
#pragma unroll
        for(int i = 0; i < 16; i += 4) {
            v2i w;
            w[0] = (int)float2_to_half2_bits_2step(o[b][i] * inv, o[b][i + 1] * inv);
            w[1] = (int)float2_to_half2_bits_2step(o[b][i + 2] * inv, o[b][i + 3] * inv);
            *reinterpret_cast<v2i*>(out + 32 * b + 8 * (i / 4) + 4 * half) = w;
        }
}

} // namespace
} // namespace w8a8
