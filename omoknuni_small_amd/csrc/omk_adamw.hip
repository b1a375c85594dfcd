// AdamW over many tensors at once, with moments in 32 bits or in 8 (include/omk_learn.h).
#include "omk_device.h"
#include "omk_learn_device.h"
#include "omk_learn_internal.h"

namespace omk {

constexpr int kAdamBlock = 256;

// Mixes the bits of a number: xorshifts and products with odd constants, every input bit reaching every output bit.
__device__ __forceinline__ uint32_t mix(uint32_t h) {
    h ^= h >> 16;
    h *= 0x7FEB352Du;
    h ^= h >> 15;
    h *= 0x846CA68Bu;
    return h ^ (h >> 16);
}

// e4m3 code (without sign) of 0 <= y <= 448.  The 20 bits of a float's mantissa that the code has no room for are rounded up
// where a random number of 20 bits (the 16 that are given, times 16) carries out of them: with the probability of
// y's place between the two codes.  Codes below 2^-6 are evenly spaced as those of the binade above are, so y is
// moved up by 2^-6 there and the code back down.
__device__ __forceinline__ uint32_t code_of(float y, uint32_t random16) {
    const bool small = y < 0.015625f;
    const uint32_t bits = __float_as_uint(small ? y + 0.015625f : y);
    return ((bits + (random16 << 4)) >> 20) - (small ? 968u : 960u);
}

__device__ __forceinline__ float from_code(uint32_t code) {
    return __builtin_amdgcn_cvt_f32_fp8((int)code, 0);
}

// The scale of a block whose largest magnitude is `top`, and what its values are multiplied by to be coded.
struct BlockScale {
    float scale, inverse;
};
__device__ __forceinline__ BlockScale block_scale(float top) {
    // (2^-100: so that one over it is a number; moments that small are kept as 0)
    if (!(top > 0x1p-100f)) return {top == top ? 0.0f : top, 0.0f};
    return {top * (1.0f / 448.0f), (1.0f / top) * 448.0f};
}

struct AdamScalars {
    float b1, c1, b2, c2;       // betas and one less them
    float rate, root, decay;    // lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t), lr * weight decay
    float eps, grad_scale;
    uint32_t key;
};

// One element.  Products and sums are rounded one by one (no fused forms): what the 8-bit states are rounded from is
// then the same number on every path.
__device__ __forceinline__ float adam(const AdamScalars &k, float p, float g, float &m, float &v, float &root) {
    g *= k.grad_scale;
    m = m * k.b1 + g * k.c1;
    v = v * k.b2 + (g * g) * k.c2;
    root = sqrtf(v);
    p = p - p * k.decay;
    return p - m * k.rate / (root * k.root + k.eps);
}

template <typename P, typename G, typename C, bool EIGHT>
__global__ __launch_bounds__(kAdamBlock) void k_adamw(AdamStep s, AdamGrads grads) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const double power1 = s.count->power1 * s.beta1, power2 = s.count->power2 * s.beta2;
    const int64_t t = s.count->steps + 1;
    const double lr = s.d_lr ? (double)*s.d_lr : s.lr;
    AdamScalars k;
    k.b1 = (float)s.beta1;
    k.c1 = (float)(1.0 - s.beta1);
    k.b2 = (float)s.beta2;
    k.c2 = (float)(1.0 - s.beta2);
    k.root = (float)(1.0 / sqrt(1.0 - power2));
    k.eps = s.eps;
    k.grad_scale = s.d_grad_scale ? *s.d_grad_scale : 1.0f;
    k.key = mix(s.seed ^ ((uint32_t)t * 0x9E3779B1u));
    for (int64_t c = blockIdx.x; c < s.n_chunks; c += gridDim.x) {
        const AdamChunk chunk = s.chunks[c];
        const G *grad = (const G *)grads.g[chunk.tensor - s.first_tensor];
        if (!grad) continue;
        const AdamTensor &a = s.tensors[chunk.tensor];
        k.rate = (float)(lr * (double)a.lr_scale / (1.0 - power1));
        k.decay = (float)(lr * (double)a.lr_scale * (double)a.weight_decay);
        for (int u = wave; u < kChunkUnits; u += kAdamBlock / 64) {
            const int64_t unit = (int64_t)chunk.chunk * kChunkUnits + u;
            const int64_t base = unit * kUnit;
            if (base >= a.n) break;
            float m[4], v[4], root[4];
            // largest magnitudes as bit patterns: these have the numbers' order, with NaN above all of them
            uint32_t top_m = 0, top_v = 0;
            const float scale_m = EIGHT ? a.m_scale[unit] : 0.0f, scale_v = EIGHT ? a.v_scale[unit] : 0.0f;
            for (int i = 0; i < 4; i++) {
                const int64_t at = base + lane * 4 + i;
                m[i] = v[i] = root[i] = 0.0f;
                if (at >= a.n) continue;
                if (EIGHT) {
                    m[i] = from_code(((const uint8_t *)a.m)[at]) * scale_m;
                    const float r = from_code(((const uint8_t *)a.v)[at]) * scale_v;
                    v[i] = r * r;
                } else {
                    m[i] = ((const float *)a.m)[at];
                    v[i] = ((const float *)a.v)[at];
                }
                const float p = adam(k, (float)((const P *)a.param)[at], (float)grad[at], m[i], v[i], root[i]);
                ((P *)a.param)[at] = (P)p;
                if (a.copy) ((C *)a.copy)[at] = (C)p;
                if (!EIGHT) {
                    ((float *)a.m)[at] = m[i];
                    ((float *)a.v)[at] = v[i];
                }
                top_m = umax32(top_m, __float_as_uint(fabsf(m[i])));
                top_v = umax32(top_v, __float_as_uint(fabsf(root[i])));
            }
            if (!EIGHT) continue;
            const BlockScale sm = block_scale(__uint_as_float(wave_max_all(top_m)));
            const BlockScale sv = block_scale(__uint_as_float(wave_max_all(top_v)));
            if (lane == 0) {
                a.m_scale[unit] = sm.scale;
                a.v_scale[unit] = sv.scale;
            }
            const uint32_t key = mix(k.key ^ (uint32_t)(a.first_unit + unit));
            for (int i = 0; i < 4; i++) {
                const int64_t at = base + lane * 4 + i;
                if (at >= a.n) continue;
                const uint32_t random = mix(key + (uint32_t)(lane * 4 + i) * 0x9E3779B1u);
                const float ym = fminf(fabsf(m[i]) * sm.inverse, 448.0f), yv = fminf(root[i] * sv.inverse, 448.0f);
                uint32_t cm = code_of(ym, random & 0xFFFFu), cv = code_of(yv, random >> 16);
                if (yv > 0.0f && cv == 0) cv = 1;
                if (m[i] < 0.0f) cm |= 0x80u;
                ((uint8_t *)a.m)[at] = (uint8_t)cm;
                ((uint8_t *)a.v)[at] = (uint8_t)cv;
            }
        }
    }
    if (!s.last) return;
    // The last block to come here counts the step: all others have read the count.
    __syncthreads();
    if (threadIdx.x) return;
    __threadfence();
    if (atomicAdd(&s.count->done, 1u) != gridDim.x - 1) return;
    s.count->power1 = power1;
    s.count->power2 = power2;
    s.count->steps = t;
    s.count->done = 0;
}

__global__ void k_adamw_set(AdamCount *count, int64_t steps, double power1, double power2) {
    count->power1 = power1;
    count->power2 = power2;
    count->steps = steps;
    count->done = 0;
}

hipError_t launch_adamw_set(AdamCount *count, int64_t steps, double power1, double power2, hipStream_t stream) {
    k_adamw_set<<<1, 1, 0, stream>>>(count, steps, power1, power2);
    return hipGetLastError();
}

// Blocks of a launch at most: each takes chunks in turn, so that the count of blocks done stays one counter.
constexpr int64_t kAdamGrid = 2048;

template <typename P, typename G, typename C>
static hipError_t launch(int state, const AdamStep &s, const AdamGrads &g, hipStream_t stream) {
    const dim3 grid((unsigned)(s.n_chunks < 1 ? 1 : s.n_chunks < kAdamGrid ? s.n_chunks : kAdamGrid));
    if (state == OMK_F8)
        k_adamw<P, G, C, true><<<grid, kAdamBlock, 0, stream>>>(s, g);
    else
        k_adamw<P, G, C, false><<<grid, kAdamBlock, 0, stream>>>(s, g);
    return hipGetLastError();
}

template <typename G>
static hipError_t launch_f32(int copy, int state, const AdamStep &s, const AdamGrads &g, hipStream_t stream) {
    return copy == OMK_F16 ? launch<float, G, f16_t>(state, s, g, stream) : launch<float, G, bf16_t>(state, s, g, stream);
}

hipError_t launch_adamw(int param, int grad, int copy, int state, const AdamStep &s, const AdamGrads &g,
                        hipStream_t stream) {
    if (param == OMK_F32) {
        if (grad == OMK_F32) return launch_f32<float>(copy, state, s, g, stream);
        if (grad == OMK_BF16) return launch_f32<bf16_t>(copy, state, s, g, stream);
        return launch_f32<f16_t>(copy, state, s, g, stream);
    }
    if (param == OMK_BF16) {
        if (grad == OMK_F32) return launch<bf16_t, float, bf16_t>(state, s, g, stream);
        return launch<bf16_t, bf16_t, bf16_t>(state, s, g, stream);
    }
    if (grad == OMK_F32) return launch<f16_t, float, f16_t>(state, s, g, stream);
    return launch<f16_t, f16_t, f16_t>(state, s, g, stream);
}

}  // namespace omk
