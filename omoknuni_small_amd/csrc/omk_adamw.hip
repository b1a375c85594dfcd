// AdamW over many tensors at once, with moments in 32 bits or in 8 (include/omk_learn.h).
#include "omk_device.h"
#include "omk_learn_device.h"
#include "omk_learn_internal.h"

namespace omk {

constexpr int kAdamBlock = 256;

// Mixes the bits of a number: the published 32-bit integer hash "lowbias32" (C. Wellons, 2018), its shifts and constants.
__device__ __forceinline__ uint32_t mix(uint32_t h) {
    h ^= h >> 16;
    h *= 0x7FEB352Du;
    h ^= h >> 15;
    h *= 0x846CA68Bu;
    return h ^ (h >> 16);
}

// The e4m3 code of |y| <= 448, put into byte AT of `codes`: the 20 bits of the float's mantissa that the code has no room for
// (counted from 2^-9 upwards where codes are evenly spaced, below 2^-6) are rounded up where the random number's upper 20
// bits carry out of them, with the probability of y's place between the two codes.  One instruction
// (v_cvt_sr_fp8_f32); from the definition, by integer operations, it took fourteen.
template <int AT>
__device__ __forceinline__ uint32_t put_code(uint32_t codes, float y, uint32_t random) {
    return (uint32_t)__builtin_amdgcn_cvt_sr_fp8_f32(y, (int)random, (int)codes, AT);
}

template <int AT>
__device__ __forceinline__ float from_code(uint32_t codes) {
    return __builtin_amdgcn_cvt_f32_fp8((int)codes, AT);
}
// Four codes of a word as floats, and back.
__device__ __forceinline__ void from_codes(uint32_t codes, float scale, float (&x)[4]) {
    x[0] = from_code<0>(codes) * scale;
    x[1] = from_code<1>(codes) * scale;
    x[2] = from_code<2>(codes) * scale;
    x[3] = from_code<3>(codes) * scale;
}
__device__ __forceinline__ uint32_t to_codes(const float (&x)[4], float inverse, const uint32_t (&random)[4]) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = __builtin_amdgcn_fmed3f(x[i] * inverse, -448.0f, 448.0f);
    uint32_t codes = put_code<0>(0u, y[0], random[0]);
    codes = put_code<1>(codes, y[1], random[1]);
    codes = put_code<2>(codes, y[2], random[2]);
    return put_code<3>(codes, y[3], random[3]);
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

// powers: beta^(steps + 1)
__device__ __forceinline__ void count_of(AdamCount *count, int64_t steps, double power1, double power2) {
    count->power1 = power1;
    count->power2 = power2;
    count->unbias = 1.0 / (1.0 - power1);
    count->root = (float)(1.0 / sqrt(1.0 - power2));
    count->steps = steps;
    count->done = 0;
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
    // (a reciprocal good to a unit in the last place and a product: the quotient rounded once would be nine instructions more)
    return p - m * k.rate * __builtin_amdgcn_rcpf(root * k.root + k.eps);
}

template <bool EIGHT>
struct State {
    typedef float type;
};
template <>
struct State<true> {
    typedef uint8_t type;
};

// Tensors' addresses come from memory, where the compiler cannot tell what they address: device memory, all of them.
template <typename T>
using Global = __attribute__((address_space(1))) T;

// Four neighbouring elements of a tensor, which a lane takes: WHOLE = as one vector, else as many as there are, one by one.
template <typename T>
struct alignas(4 * sizeof(T)) Four {
    T x[4];
};
__device__ __forceinline__ float read_lane(float v, int lane) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}

template <bool WHOLE, typename T>
__device__ __forceinline__ Four<T> load4(const void *from, int64_t base, int lane, int there) {
    typedef uint32_t Raw __attribute__((ext_vector_type(sizeof(T))));
    union {
        Four<T> f;
        Raw raw;
    } u;
    const Global<const T> *at = (const Global<const T> *)from + base;
    if (WHOLE) {
        u.raw = __builtin_nontemporal_load((const Global<const Raw> *)at + lane);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) u.f.x[i] = i < there ? at[4 * lane + i] : T(0);
    }
    return u.f;
}
template <bool WHOLE, typename T>
__device__ __forceinline__ void store4(void *to, int64_t base, int lane, int there, const Four<T> &f) {
    typedef uint32_t Raw __attribute__((ext_vector_type(sizeof(T))));
    union {
        Four<T> f;
        Raw raw;
    } u;
    u.f = f;
    Global<T> *at = (Global<T> *)to + base;
    if (WHOLE) {
        __builtin_nontemporal_store(u.raw, (Global<Raw> *)at + lane);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i < there) at[4 * lane + i] = u.f.x[i];
    }
}

// A thread takes four elements, a wavefront a unit of 256, kUnitsAtOnce of them at a time: what bounds the step is memory's rate,
// and with it the loads on their way.  95 M weights with bf16 gradients and copies: 492 us with 32-bit moments (28 bytes a
// weight, 5.4 TB/s), 348 us with 8-bit ones (16 bytes, 4.4 TB/s); with two units at once 527 and 412 us, with eight 521 and 384 us.
constexpr int kUnitsAtOnce = 4;

// COUNT units of a tensor from `unit` on; all loads are on their way before the first is needed.  WHOLE: all their elements are
// there, at addresses that vectors can be taken from.
template <typename P, typename G, typename C, bool EIGHT, bool WHOLE, int COUNT>
__device__ __forceinline__ void step_units(const AdamScalars &k, const AdamTensor &a, const G *grad, int64_t unit, int lane) {
    typedef typename State<EIGHT>::type S;
    const int64_t base = unit * kUnit;
    const int there = WHOLE ? 4 : (int)max((int64_t)0, min((int64_t)4, a.n - base - 4 * lane));
    Four<P> p[COUNT];
    Four<G> g[COUNT];
    Four<S> m[COUNT], v[COUNT];
    // (lane u holds unit u's scales)
    Global<float> *m_scale = (Global<float> *)a.m_scale + unit, *v_scale = (Global<float> *)a.v_scale + unit;
    float scale_m = 0.0f, scale_v = 0.0f;
    if (EIGHT && lane < COUNT) {
        scale_m = m_scale[lane];
        scale_v = v_scale[lane];
    }
#pragma unroll
    for (int u = 0; u < COUNT; u++) {
        p[u] = load4<WHOLE, P>(a.param, base + u * kUnit, lane, there);
        g[u] = load4<WHOLE, G>(grad, base + u * kUnit, lane, there);
        m[u] = load4<WHOLE, S>(a.m, base + u * kUnit, lane, there);
        v[u] = load4<WHOLE, S>(a.v, base + u * kUnit, lane, there);
    }
#pragma unroll
    for (int u = 0; u < COUNT; u++) {
        float fm[4], root[4];
        Four<C> copy;
        // largest magnitudes as bit patterns: these have the numbers' order, with NaN above all of them
        uint32_t top_m = 0, top_v = 0;
        if constexpr (EIGHT) {
            from_codes(__builtin_bit_cast(uint32_t, m[u]), read_lane(scale_m, u), fm);
            from_codes(__builtin_bit_cast(uint32_t, v[u]), read_lane(scale_v, u), root);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float fv;
            if constexpr (EIGHT) {
                fv = root[i] * root[i];
            } else {
                fm[i] = m[u].x[i];
                fv = v[u].x[i];
            }
            const float np = adam(k, (float)p[u].x[i], (float)g[u].x[i], fm[i], fv, root[i]);
            p[u].x[i] = (P)np;
            copy.x[i] = (C)np;
            if constexpr (EIGHT) {
                top_m = umax32(top_m, __float_as_uint(fabsf(fm[i])));
                top_v = umax32(top_v, __float_as_uint(fabsf(root[i])));
            } else {
                m[u].x[i] = fm[i];
                v[u].x[i] = fv;
            }
        }
        store4<WHOLE, P>(a.param, base + u * kUnit, lane, there, p[u]);
        if (a.copy) store4<WHOLE, C>(a.copy, base + u * kUnit, lane, there, copy);
        if constexpr (EIGHT) {
            const BlockScale sm = block_scale(__uint_as_float(wave_max_all(top_m)));
            const BlockScale sv = block_scale(__uint_as_float(wave_max_all(top_v)));
            if (lane == u) {
                scale_m = sm.scale;
                scale_v = sv.scale;
            }
            const uint32_t key = mix(k.key ^ (uint32_t)(a.first_unit + unit + u));
            uint32_t for_m[4], for_v[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t random = mix(key + (uint32_t)(lane * 4 + i) * 0x9E3779B1u);
                for_m[i] = random << 16;
                for_v[i] = random & 0xFFFF0000u;
            }
            m[u] = __builtin_bit_cast(Four<S>, to_codes(fm, sm.inverse, for_m));
            uint32_t codes = to_codes(root, sv.inverse, for_v);
            // what is not nothing is not kept as nothing: the smallest code in the place of 0
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (root[i] * sv.inverse > 0.0f && (codes >> 8 * i & 0xFFu) == 0) codes |= 1u << 8 * i;
            v[u] = __builtin_bit_cast(Four<S>, codes);
        }
        store4<WHOLE, S>(a.m, base + u * kUnit, lane, there, m[u]);
        store4<WHOLE, S>(a.v, base + u * kUnit, lane, there, v[u]);
    }
    if (EIGHT && lane < COUNT) {
        m_scale[lane] = scale_m;
        v_scale[lane] = scale_v;
    }
}

template <typename P, typename G, typename C, bool EIGHT>
__global__ __launch_bounds__(kAdamBlock) void k_adamw(AdamStep s, AdamGrads grads) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const double unbias = s.count->unbias, lr = s.d_lr ? (double)*s.d_lr : s.lr;
    AdamScalars k;
    k.b1 = (float)s.beta1;
    k.c1 = (float)(1.0 - s.beta1);
    k.b2 = (float)s.beta2;
    k.c2 = (float)(1.0 - s.beta2);
    k.root = s.count->root;
    k.eps = s.eps;
    k.grad_scale = s.d_grad_scale ? *s.d_grad_scale : 1.0f;
    k.key = mix(s.seed ^ (uint32_t)(s.count->steps + 1) * 0x9E3779B1u);
    for (int64_t c = blockIdx.x; c < s.n_chunks; c += gridDim.x) {
        const AdamChunk chunk = s.chunks[c];
        const G *grad = (const G *)grads.g[chunk.tensor - s.first_tensor];
        if (!grad) continue;
        const AdamTensor &a = s.tensors[chunk.tensor];
        k.rate = (float)(lr * (double)a.lr_scale * unbias);
        k.decay = (float)(lr * (double)a.lr_scale * (double)a.weight_decay);
        const int64_t begin = (int64_t)chunk.chunk * s.chunk_units, end = min(begin + s.chunk_units, (a.n + kUnit - 1) / kUnit);
        const bool vectors = a.vectors && ((uintptr_t)grad & (4 * sizeof(G) - 1)) == 0;
        // chunks of few units: one for a wavefront
        const int at_once = s.chunk_units < kUnitsAtOnce * (kAdamBlock / 64) ? 1 : kUnitsAtOnce;
        for (int64_t unit = begin + wave * at_once; unit < end; unit += at_once * (kAdamBlock / 64)) {
            if (at_once > 1 && vectors && (unit + kUnitsAtOnce) * kUnit <= a.n) {
                step_units<P, G, C, EIGHT, true, kUnitsAtOnce>(k, a, grad, unit, lane);
                continue;
            }
            for (int64_t u = unit; u < min(unit + at_once, end); u++) {
                if (vectors && (u + 1) * kUnit <= a.n)
                    step_units<P, G, C, EIGHT, true, 1>(k, a, grad, u, lane);
                else
                    step_units<P, G, C, EIGHT, false, 1>(k, a, grad, u, lane);
            }
        }
    }
    if (!s.last) return;
    // The last block to come here counts the step (the last of its group first: 480 blocks that all counted at one address took
    // 7 us for it, 14 ns each): whatever the others take from the count they have taken before the
    // barrier.  (Nothing else is handed over, so no fence, which would write the caches back in every block.)
    __syncthreads();
    if (threadIdx.x) return;
    const uint32_t group = blockIdx.x % kCountGroups, groups = min(gridDim.x, (uint32_t)kCountGroups);
    uint32_t *done = s.done + group * kCountStep;
    if (atomicAdd(done, 1u) != (gridDim.x - group + kCountGroups - 1) / kCountGroups - 1) return;
    *done = 0;
    if (atomicAdd(&s.count->done, 1u) != groups - 1) return;
    count_of(s.count, s.count->steps + 1, s.count->power1 * s.beta1, s.count->power2 * s.beta2);
}

__global__ __launch_bounds__(kCountGroups) void k_adamw_set(AdamCount *count, uint32_t *done, int64_t steps, double power1,
                                                            double power2) {
    done[threadIdx.x * kCountStep] = 0;
    if (threadIdx.x == 0) count_of(count, steps, power1, power2);
}

hipError_t launch_adamw_set(AdamCount *count, uint32_t *done, int64_t steps, double power1, double power2, hipStream_t stream) {
    k_adamw_set<<<1, kCountGroups, 0, stream>>>(count, done, steps, power1, power2);
    return hipGetLastError();
}

// Blocks of a launch at most.  One chunk a block, up to there: 95 M weights with 8-bit moments take 348 us so, and 369 us with 2048
// blocks that take chunks in turn, whose last turn only some of them have.
constexpr int64_t kAdamGrid = 16384;

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
