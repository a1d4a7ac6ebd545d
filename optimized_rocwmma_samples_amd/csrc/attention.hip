// attention.hip -- causal attention of whole prompts for gfx950.
#include "w8a8_device.hpp"
#include "w8a8_internal.hpp"

namespace w8a8 {
namespace {

// One wave per (token, head): lanes over the channels, one key after the other
// with a running maximum and sum.
template <int D>
__global__ void __launch_bounds__(kWave) attention_kernel(AttentionArgs a)
{
    constexpr int  kC   = D / kWave;
    const uint32_t head = blockIdx.x % a.heads, t = blockIdx.x / a.heads, lane = threadIdx.x;
    const uint32_t kvh  = head / (a.heads / a.kv_heads);
    // the last sequence that starts at or before t
    uint32_t lo = 0, hi = a.seqs;
    while(hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if(a.starts[mid] <= (int32_t)t)
            lo = mid;
        else
            hi = mid;
    }
    const int32_t begin = max(a.starts[lo], 0);
    if(begin > (int32_t)t || a.starts[lo + 1] <= (int32_t)t) return;
    float q[kC], o[kC];
#pragma unroll
    for(int i = 0; i < kC; ++i) {
        q[i] = half_bits_to_float(a.q[(size_t)t * a.ldq + head * D + lane * kC + i]) * a.scale;
        o[i] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for(uint32_t j = begin; j <= t; ++j) {
        float dot = 0.f;
#pragma unroll
        for(int i = 0; i < kC; ++i)
            dot = fmaf(q[i], half_bits_to_float(a.k[(size_t)j * a.ldk + kvh * D + lane * kC + i]), dot);
        const float s  = wave_sum(dot);
        const float mn = fmaxf(m, s);
        const float al = m == mn ? 1.f : __expf(m - mn), p = s == mn ? 1.f : __expf(s - mn);
        m              = mn;
        l              = l * al + p;
#pragma unroll
        for(int i = 0; i < kC; ++i)
            o[i] = o[i] * al + p * half_bits_to_float(a.v[(size_t)j * a.ldv + kvh * D + lane * kC + i]);
    }
#pragma unroll
    for(int i = 0; i < kC; ++i)
        a.out[(size_t)t * a.ldo + head * D + lane * kC + i] = float_to_half_bits(o[i] / l);
}

} // namespace

hipError_t launch_attention(const AttentionArgs& a, hipStream_t stream)
{
    if(a.dim == 64)
        attention_kernel<64><<<a.tokens * a.heads, kWave, 0, stream>>>(a);
    else
        attention_kernel<128><<<a.tokens * a.heads, kWave, 0, stream>>>(a);
    return hipGetLastError();
}

} // namespace w8a8
