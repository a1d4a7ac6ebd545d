// moe_route.hpp -- the routing of one token by one wave, shared by the kernels
// that route (moe.hip, moe_decode.hip): the same order of operations in each,
// so the ids and weights are the same bits.
#pragma once

#include "w8a8_device.hpp"

namespace w8a8 {

// Element i of logits held as fp16 or fp32.
template <bool F16>
__device__ __forceinline__ float load_logit(const void* p, size_t i)
{
    if constexpr(F16)
        return half_bits_to_float(static_cast<const uint16_t*>(p)[i]);
    else
        return static_cast<const float*>(p)[i];
}

// (value, index) of the better of two candidates: larger value, then lower index.
__device__ __forceinline__ void better(float& v, int& i, float ov, int oi)
{
    if(ov > v || (ov == v && oi < i)) {
        v = ov;
        i = oi;
    }
}

// The topk experts of one token, best first: emit(k, id, weight) in every lane
// for k = 0 .. topk - 1, id = -1 and weight = 0 where only NaN logits are left; one NaN
// makes the sum NaN and with it every weight 0.
// Experts are chosen on the logits (softmax is monotonic, so the choice is
// exact), the lower index winning ties; weight = exp(l - max) * (1 / sum_e
// exp(l_e - max)).  logit(e): the fp32 value of expert e's logit.  A lane owns
// experts lane, lane + 64, ...: experts <= 4096 (the bits of `used`).  HELD > 0:
// they are read once into that many registers (experts <= 64 * HELD), instead of
// again for every pick.
template <int HELD, class Logit, class Emit>
__device__ __forceinline__ void route_token_held(Logit logit, uint32_t experts, uint32_t topk,
                                                 int lane, Emit emit)
{
    float held[HELD > 0 ? HELD : 1];
    // each(f): f(j, expert, its logit) over the lane's experts in ascending order
    auto each = [&](auto f) {
        if constexpr(HELD > 0) {
#pragma unroll
            for(int j = 0; j < HELD; ++j) {
                const uint32_t e = lane + j * kWave;
                if(e < experts) f(j, e, held[j]);
            }
        } else {
            int j = 0;
            for(uint32_t e = lane; e < experts; e += kWave, ++j) f(j, e, logit(e));
        }
    };
    if constexpr(HELD > 0)
#pragma unroll
        for(int j = 0; j < HELD; ++j)
            held[j] = lane + j * kWave < experts ? logit(lane + j * kWave) : 0.f;

    // cross-lane steps are DPP reductions (no LDS round trips)
    float wmax = -INFINITY;
    each([&](int, uint32_t, float v) { wmax = fmaxf(wmax, v); });
    wmax       = wave_max(wmax);
    float wsum = 0.f;
    each([&](int, uint32_t, float v) { wsum += expf(v - wmax); });
    wsum            = wave_sum(wsum);
    const float inv = wsum > 0.f ? 1.f / wsum : 0.f;

    // `used` marks the chosen ones.  Per pick: each lane's best unused candidate
    // (larger logit, then lower index), the wave max of those values, then the
    // lowest index among the lanes holding that max: the same winner as a
    // pairwise reduction.
    constexpr int kNone = 0x7FFFFFFF;
    uint64_t      used  = 0;
    for(uint32_t k = 0; k < topk; ++k) {
        float bv = -INFINITY;
        int   bi = kNone;
        each([&](int j, uint32_t e, float v) {
            if(!((used >> j) & 1u)) better(bv, bi, v, (int)e);
        });
        const float m = wave_max(bv);
        const int   w = wave_min_i32(bv == m ? bi : kNone);
        if(w != kNone && (uint32_t)w % kWave == (uint32_t)lane) used |= 1ull << ((uint32_t)w / kWave);
        const bool ok = w != kNone;
        emit(k, ok ? w : -1, ok ? expf(m - wmax) * inv : 0.f);
    }
}

template <class Logit, class Emit>
__device__ __forceinline__ void route_token(Logit logit, uint32_t experts, uint32_t topk, int lane,
                                            Emit emit)
{
    if(experts <= kWave)
        route_token_held<1>(logit, experts, topk, lane, emit);
    else if(experts <= 4 * kWave)
        route_token_held<4>(logit, experts, topk, lane, emit);
    else
        route_token_held<0>(logit, experts, topk, lane, emit);
}

} // namespace w8a8
