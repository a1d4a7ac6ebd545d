// kv4_device.hpp -- what the kernels of the paged 4-bit cache share.
#pragma once

#include "matrix_f16.hpp"
#include "w8a8_internal.hpp"

#include <type_traits>

namespace w8a8 {
namespace {

struct CacheView {
    uint8_t*  codes[2];  // keys, values
    uint32_t* scales[2]; // (scale, offset) fp16 pairs
    uint32_t  slots;     // pages * page_size
    uint32_t  page_shift, page_size, kv_heads;
};

CacheView view(const w8a8_kv4_cache& c)
{
    return {{c.k_codes, c.v_codes},
            {static_cast<uint32_t*>(c.k_scales), static_cast<uint32_t*>(c.v_scales)},
            c.pages * c.page_size,
            (uint32_t)__builtin_ctz(c.page_size),
            c.page_size,
            c.kv_heads};
}

// Row number of (page, head, place) in the codes and scales.
__device__ __forceinline__ size_t cache_row(const CacheView& c, uint32_t page, uint32_t head,
                                            uint32_t place)
{
    return ((size_t)page * c.kv_heads + head) * c.page_size + place;
}

// Two fp32 results as packed fp16, those past its range as its ends: the last code of a
// group that reaches 65504 may stand for a little more, its step being rounded (0 .. 65504
// has steps of 4368 and ends at 65520, which would be an infinity).  NaN stays NaN.
__device__ __forceinline__ uint32_t finite_halves(float a, float b)
{
    const v2h most = {(_Float16)65504.f, (_Float16)65504.f};
    const v2h h    = __builtin_bit_cast(v2h, float2_to_half2_bits_2step(a, b));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_minimum(
                                            __builtin_elementwise_maximum(h, -most), most));
}

// N dwords, N = 1, 2 or 4, from global memory in one access.
template <int N>
__device__ __forceinline__ void load_dwords(int32_t* r, const void* p)
{
    if constexpr(N == 4) {
        const v4i u = *static_cast<const v4i*>(p);
#pragma unroll
        for(int i = 0; i < 4; ++i) r[i] = u[i];
    } else if constexpr(N == 2) {
        const v2i u = *static_cast<const v2i*>(p);
        r[0] = u[0];
        r[1] = u[1];
    } else
        r[0] = *static_cast<const int32_t*>(p);
}

// v and the sum of v over the lanes before.
__device__ __forceinline__ uint32_t lanes_sum(uint32_t v)
{
    const auto add = [&](auto ctrl, auto rows) {
        v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value,
                                                   decltype(rows)::value, 0xF, false);
    };
    using std::integral_constant;
    add(integral_constant<int, 0x111>(), integral_constant<int, 0xF>()); // from 1, 2, 4, 8 lanes
    add(integral_constant<int, 0x112>(), integral_constant<int, 0xF>()); // before, in rows of 16
    add(integral_constant<int, 0x114>(), integral_constant<int, 0xF>());
    add(integral_constant<int, 0x118>(), integral_constant<int, 0xF>());
    add(integral_constant<int, 0x142>(), integral_constant<int, 0xA>()); // the row before's last
    add(integral_constant<int, 0x143>(), integral_constant<int, 0xC>()); // lane 31's
    return v;
}

// The instantiation for a cache's head width and group.
template <class F>
void with_widths(const w8a8_kv4_cache& c, F f)
{
    using std::integral_constant;
    if(c.head_dim == 64) {
        if(c.group == 32)
            f(integral_constant<int, 64>(), integral_constant<int, 32>());
        else
            f(integral_constant<int, 64>(), integral_constant<int, 64>());
    } else {
        if(c.group == 32)
            f(integral_constant<int, 128>(), integral_constant<int, 32>());
        else if(c.group == 64)
            f(integral_constant<int, 128>(), integral_constant<int, 64>());
        else
            f(integral_constant<int, 128>(), integral_constant<int, 128>());
    }
}

} // namespace
} // namespace w8a8
