// Device-side building blocks of the operators behind include/omk_learn.h.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace omk {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

constexpr float kLog2E = 1.44269504088896341f;
constexpr double kLn2 = 0.693147180559945309417;

// exp(x) of a difference to the row's largest logit: one product and v_exp_f32 (2^x, good to a unit in the last place).
// The product's rounding makes exp(x) off by |x| 2^-24 relative: nothing where the value counts, since it is
// exp(x) itself that gets small.  Below 2^-126 the result may be flushed to 0: 1e-38 of the largest term.
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2E); }

// log(s) in 64 bits from a 32-bit sum: the exponent is taken off, so that what is rounded is the logarithm of a number
// near 1.  (A loss compares a ratio with borders: the log-probability keeps more than the 24 bits of one float.)
__device__ __forceinline__ double log_of_sum(float s) {
    int k = __builtin_amdgcn_frexp_expf(s);
    float f = __builtin_amdgcn_frexp_mantf(s);  // [0.5, 1)
    if (f < 0.70710678f) {
        f *= 2.0f;
        k--;
    }
    return (double)k * kLn2 + (double)logf(f);
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}

// What a row comes to: largest legal logit, sum of exp(x - top) over the legal ones (0: no policy), sum of
// exp(x - top) (x - top).
struct RowStats {
    float top, sum, centred;
};

}  // namespace omk
