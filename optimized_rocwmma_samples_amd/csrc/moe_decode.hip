// moe_decode.hip -- the expert layer of the few tokens of a decode step for
// gfx950, in two launches.
#include "moe_route.hpp"
#include "w8a8_device.hpp"
#include "w8a8_internal.hpp"

namespace w8a8 {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves   = kThreads / kWave;

// Workspace: the activations of the pairs, then their experts and weights.
struct Ws {
    float*   act;    // [pairs, inter]
    int32_t* ids;    // [pairs]
    float*   weight; // [pairs]
};

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

Ws carve(const MoeDecodeArgs& a)
{
    uint8_t* p     = static_cast<uint8_t*>(a.ws);
    const size_t n = (size_t)a.tokens * a.topk;
    Ws           w;
    w.act = reinterpret_cast<float*>(p);
    p += up256(n * a.inter * 4);
    w.ids = reinterpret_cast<int32_t*>(p);
    p += up256(n * 4);
    w.weight = reinterpret_cast<float*>(p);
    return w;
}

__device__ __forceinline__ float block_max(float v, float* red)
{
    v = wave_max(v);
    __syncthreads();
    if(threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = v;
    __syncthreads();
    float m = red[0];
    for(int i = 1; i < kWaves; ++i) m = fmaxf(m, red[i]);
    return m;
}

// Sum over k of w[k] * q[k] by one wave, n a multiple of 16.
__device__ __forceinline__ int dot_i8(const int8_t* w, const int8_t* q, uint32_t n, int lane)
{
    int acc = 0;
    for(uint32_t k = lane * 16; k < n; k += kWave * 16) {
        const v4i a = *reinterpret_cast<const v4i*>(w + k);
        const v4i b = *reinterpret_cast<const v4i*>(q + k);
#pragma unroll
        for(int i = 0; i < 4; ++i) acc = __builtin_amdgcn_sdot4(a[i], b[i], acc, false);
    }
    for(int d = 32; d > 0; d >>= 1) acc += __shfl_xor(acc, d, kWave);
    return acc;
}

template <bool F16>
__global__ void __launch_bounds__(kThreads) gate_up_kernel(MoeDecodeArgs a, Ws ws)
{
    extern __shared__ int8_t q[]; // [hidden]
    __shared__ float         red[kWaves];
    __shared__ int           s_id;
    const uint32_t pair = blockIdx.y, t = pair / a.topk, slot = pair % a.topk;
    const int      lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    if(wave == 0)
        route_token([&](uint32_t e) { return load_logit<F16>(a.logits, (size_t)t * a.experts + e); },
                    a.experts, slot + 1, lane, [&](uint32_t k, int id, float w) {
                        if(k == slot && lane == 0) {
                            s_id = id;
                            if(blockIdx.x == 0) {
                                ws.ids[pair]    = id;
                                ws.weight[pair] = w;
                            }
                        }
                    });
    __syncthreads();
    const int e = s_id;
    if(e < 0) return;
    const uint16_t* x = a.x + (size_t)t * a.ldx;
    const float*    s = a.s + (size_t)e * a.hidden;
    float           m = 0.f;
    for(uint32_t k = threadIdx.x; k < a.hidden; k += kThreads)
        m = fmaxf(m, fabsf(half_bits_to_float(x[k]) * s[k]));
    m               = block_max(m, red);
    const float r   = m / a.qmax;
    const float inv = r > 0.f ? 1.f / r : 0.f;
    for(uint32_t k = threadIdx.x; k < a.hidden; k += kThreads)
        q[k] = (int8_t)quant_i8(half_bits_to_float(x[k]) * s[k], inv, a.qmax);
    __syncthreads();
    for(uint32_t j = blockIdx.x * kWaves + wave; j < a.inter; j += gridDim.x * kWaves) {
        const size_t row = (size_t)e * 2 * a.inter + j;
        const int    ag  = dot_i8(a.wgu + row * a.hidden, q, a.hidden, lane);
        const int    au  = dot_i8(a.wgu + (row + a.inter) * a.hidden, q, a.hidden, lane);
        const float  g   = ((float)ag * r) * a.sgu[row];
        const float  u   = ((float)au * r) * a.sgu[row + a.inter];
        float        h   = silu_mul(g, u);
        if(a.s2) h *= a.s2[(size_t)e * a.inter + j];
        if(lane == 0) ws.act[(size_t)pair * a.inter + j] = h;
    }
}

__global__ void __launch_bounds__(kThreads) down_kernel(MoeDecodeArgs a, Ws ws)
{
    extern __shared__ int8_t q[]; // [inter]
    __shared__ float         red[kWaves];
    const uint32_t t = blockIdx.y;
    const int      lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const uint32_t j   = blockIdx.x * kWaves + wave;
    float          acc = 0.f;
    for(uint32_t slot = 0; slot < a.topk; ++slot) {
        const uint32_t pair = t * a.topk + slot;
        const int      e    = ws.ids[pair];
        if(e < 0) continue;
        const float* h = ws.act + (size_t)pair * a.inter;
        float        m = 0.f;
        for(uint32_t k = threadIdx.x; k < a.inter; k += kThreads) m = fmaxf(m, fabsf(h[k]));
        m               = block_max(m, red);
        const float r   = m / a.qmax;
        const float inv = r > 0.f ? 1.f / r : 0.f;
        for(uint32_t k = threadIdx.x; k < a.inter; k += kThreads)
            q[k] = (int8_t)quant_i8(h[k], inv, a.qmax);
        __syncthreads();
        if(j < a.hidden) {
            const size_t row = (size_t)e * a.hidden + j;
            const int    d   = dot_i8(a.wd + row * a.inter, q, a.inter, lane);
            acc              = fmaf(ws.weight[pair], ((float)d * r) * a.sd[row], acc);
        }
        __syncthreads();
    }
    if(j < a.hidden && lane == 0) a.out[(size_t)t * a.ldo + j] = float_to_half_bits(acc);
}

} // namespace

size_t moe_ffn_decode_workspace_bytes(uint32_t tokens, uint32_t topk, uint32_t hidden, uint32_t inter)
{
    const size_t n = (size_t)tokens * topk;
    return up256(n * inter * 4) + 2 * up256(n * 4);
}

hipError_t launch_moe_ffn_decode(const MoeDecodeArgs& a, bool f16, hipStream_t stream)
{
    const Ws   ws = carve(a);
    const dim3 grid((a.inter + 4 * kWaves - 1) / (4 * kWaves), a.tokens * a.topk);
    if(f16)
        gate_up_kernel<true><<<grid, kThreads, a.hidden, stream>>>(a, ws);
    else
        gate_up_kernel<false><<<grid, kThreads, a.hidden, stream>>>(a, ws);
    hipError_t e = hipGetLastError();
    if(e != hipSuccess) return e;
    down_kernel<<<dim3((a.hidden + kWaves - 1) / kWaves, a.tokens), kThreads, a.inter, stream>>>(a,
                                                                                                 ws);
    return hipGetLastError();
}

} // namespace w8a8
