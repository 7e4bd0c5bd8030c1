// f32 values as sums of two f16 values, for products on the f16 matrix cores.
#pragma once
#include "common.hpp"

namespace barq {

typedef _Float16 h2v __attribute__((ext_vector_type(2)));

// x0, x1 -> packed f16 (hi) and packed f16 of what hi leaves (lo): one packed
// conversion and two v_fma_mix{lo,hi}_f16.  The empty asm keeps the compiler
// from converting every value a second time, and minus_one (-1 in a register
// it knows nothing of) from turning the fma into a conversion and a
// subtraction.
__device__ __forceinline__ float f16_minus_one() {
    float v = -1.0f;
    asm("" : "+s"(v));
    return v;
}
__device__ __forceinline__ void split_f16(float x0, float x1, float minus_one, uint32_t& hi, uint32_t& lo) {
    asm("" : "+v"(x0), "+v"(x1));
    const h2v hv = {(_Float16)x0, (_Float16)x1};
    hi = __builtin_bit_cast(uint32_t, hv);
    asm("" : "+v"(hi));
    const h2v h = __builtin_bit_cast(h2v, hi);
    const float r0 = __builtin_fmaf((float)h[0], minus_one, x0), r1 = __builtin_fmaf((float)h[1], minus_one, x1);
    const h2v r = {(_Float16)r0, (_Float16)r1};
    lo = __builtin_bit_cast(uint32_t, r);
}

}  // namespace barq
