// matrix_f16.hpp -- what the attention kernels share around v_mfma_f32_32x32x16_f16.
#pragma once

#include "w8a8_device.hpp"

namespace w8a8 {
namespace {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float    v2f __attribute__((ext_vector_type(2)));
typedef float    v16f __attribute__((ext_vector_type(16)));
typedef __fp16   v4fp16 __attribute__((ext_vector_type(4)));

typedef __attribute__((address_space(3))) v4fp16 lds_v4h_t;

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

// max(a, b, c), NaN if one is: unlike fmaxf this takes no canonicalizing steps.  (Not in
// inline asm, which the compiler does not keep apart from the matrix operations before it.)
__device__ __forceinline__ float max3(float a, float b, float c)
{
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

// The values, infinities as NaN.  Scores of a query that holds an infinity are infinities and
// NaN, and so its softmax is NaN; but -infinity is also what keys get that a row may not see.
__device__ __forceinline__ v8h infinite_to_nan(v8h v)
{
    return __builtin_elementwise_fma(v, v8h{}, v);
}

} // namespace
} // namespace w8a8
