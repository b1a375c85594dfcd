// Device-side building blocks of the operators behind include/omk_learn.h.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace omk {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

constexpr float kLog2E = 1.44269504088896341f;
constexpr float kLn2 = 0.693147180559945309f, kLn2Low = (float)(0.693147180559945309 - (double)kLn2);

// exp(x) of a difference to the row's largest logit, by 2^y of v_exp_f32 (good to a unit in the last place).  Below 2^-126 the result
// may be flushed to 0.
// FINE: what y = x log2(e) lost when it was rounded, x - y ln 2, is given back: exp(x) = 2^y (1 + (x - y ln 2)).  x is -200 at least
// (or NaN).  Where sums are added up, since a log-probability's error is what is left of a ratio, of a divergence near the
// reference and of a loss whose rows cancel.  Relative errors of a term (rms, mean) for x of -4 .. -8: 3.6e-8 and -3e-9, as expf's
// (2.6e-8, -2e-9, in twice the instructions); without the correction, 1.8e-7 and 8e-8 (the constant's own rounding, alike in
// all terms), growing with |x|: nothing for a gradient.
template <bool FINE>
__device__ __forceinline__ float exp_of(float x) {
    const float y = x * kLog2E, e = __builtin_amdgcn_exp2f(y);
    if (!FINE) return e;
    return __builtin_fmaf(e, __builtin_fmaf(-y, kLn2Low, __builtin_fmaf(-y, kLn2, x)), e);
}

// x, or `least` if that is more; NaN stays (fmaxf would drop it).
__device__ __forceinline__ float at_least(float x, float least) { return __builtin_elementwise_maximum(x, least); }

// A reduction over teams of 4 .. 64 neighbouring lanes, the result in every lane of the team: lanes of a row of 16 by quad
// swaps and mirrors, rows and halves by exchanging them.  (All 64 lanes are active where these are called.)
template <int CTRL>
__device__ __forceinline__ float dpp_f32(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
    const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xF, 0xF, true);
    const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xF, 0xF, true);
    return __hiloint2double(hi, lo);
}
struct Two {
    uint32_t a, b;
};
__device__ __forceinline__ Two swap16(uint32_t v) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return {r[0], r[1]};
}
__device__ __forceinline__ Two swap32(uint32_t v) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return {r[0], r[1]};
}

template <int TEAM>
__device__ __forceinline__ float team_max(float v) {
    v = fmaxf(v, dpp_f32<0xB1>(v));   // quad_perm [1,0,3,2]
    v = fmaxf(v, dpp_f32<0x4E>(v));   // quad_perm [2,3,0,1]
    if (TEAM > 4) v = fmaxf(v, dpp_f32<0x141>(v));  // row_half_mirror
    if (TEAM > 8) v = fmaxf(v, dpp_f32<0x140>(v));  // row_mirror
    if (TEAM > 16) {
        const Two r = swap16(__float_as_uint(v));
        v = fmaxf(__uint_as_float(r.a), __uint_as_float(r.b));
    }
    if (TEAM > 32) {
        const Two r = swap32(__float_as_uint(v));
        v = fmaxf(__uint_as_float(r.a), __uint_as_float(r.b));
    }
    return v;
}

template <int TEAM>
__device__ __forceinline__ float team_sum(float v) {
    v += dpp_f32<0xB1>(v);
    v += dpp_f32<0x4E>(v);
    if (TEAM > 4) v += dpp_f32<0x141>(v);
    if (TEAM > 8) v += dpp_f32<0x140>(v);
    if (TEAM > 16) {
        const Two r = swap16(__float_as_uint(v));
        v = __uint_as_float(r.a) + __uint_as_float(r.b);
    }
    if (TEAM > 32) {
        const Two r = swap32(__float_as_uint(v));
        v = __uint_as_float(r.a) + __uint_as_float(r.b);
    }
    return v;
}

template <int TEAM>
__device__ __forceinline__ double team_sum(double v) {
    v += dpp_f64<0xB1>(v);
    v += dpp_f64<0x4E>(v);
    if (TEAM > 4) v += dpp_f64<0x141>(v);
    if (TEAM > 8) v += dpp_f64<0x140>(v);
    if (TEAM > 16) {
        const Two lo = swap16((uint32_t)__double2loint(v)), hi = swap16((uint32_t)__double2hiint(v));
        v = __hiloint2double((int)hi.a, (int)lo.a) + __hiloint2double((int)hi.b, (int)lo.b);
    }
    if (TEAM > 32) {
        const Two lo = swap32((uint32_t)__double2loint(v)), hi = swap32((uint32_t)__double2hiint(v));
        v = __hiloint2double((int)hi.a, (int)lo.a) + __hiloint2double((int)hi.b, (int)lo.b);
    }
    return v;
}

// 16 bytes of a matrix, as numbers.
template <typename T>
struct Pack {
    static constexpr int V = 16 / (int)sizeof(T);
    union {
        uint4 raw;
        T x[V];
    };
};

}  // namespace omk
