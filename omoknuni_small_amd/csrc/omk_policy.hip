// Rows of logits: which launches an operator takes (include/omk_learn.h).  The kernels over rows: omk_policy_rows.h.
#include "omk_policy_rows.h"

namespace omk {

OMK_POLICY_TYPE(extern, float)
OMK_POLICY_TYPE(extern, bf16_t)
OMK_POLICY_TYPE(extern, f16_t)

constexpr int kSumBlock = 1024;

template <typename F>
__global__ __launch_bounds__(kSumBlock) void k_sum(const F *values, int64_t n, float *out) {
    const double s = block_sum<kSumBlock>(values, n);
    if (threadIdx.x == 0) *out = (float)s;
}

// A block for every pair of lines, half of it a line: the lines' sums, the pair's loss, and the slope of every row of theirs.
__global__ __launch_bounds__(256) void k_pairs(Rows r, PreferenceLoss p) {
    const int64_t pair = blockIdx.x, line = 2 * pair + (threadIdx.x >> 7);
    const int half = threadIdx.x & 127;
    const LineRows lines = line_rows(p, r.rows);
    const int64_t begin = lines.inside(p.line_begin[line]), end = lines.inside(p.line_begin[line + 1]);
    double s = 0.0;
    for (int64_t row = begin + half; row < end; row += 128) s += p.logprob[row];
    s = team_sum<64>(s);
    __shared__ double parts[4];
    if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = s;
    __syncthreads();
    double sums[2] = {parts[0] + parts[1], parts[2] + parts[3]};
    if (half == 0 && p.line_logprob) p.line_logprob[line] = (float)sums[threadIdx.x >> 7];
    if (p.ref_logprob) {
        sums[0] -= (double)p.ref_logprob[2 * pair];
        sums[1] -= (double)p.ref_logprob[2 * pair + 1];
    }
    // (in 64 bits: where a pair's loss is least, with smoothing, its slope is what is left of two terms)
    const double u = p.beta * (sums[0] - sums[1]);
    // log(1 + exp(-|u|)), of which both losses are made
    const double t = exp(-fabs(u)), rest = log1p(t);
    double loss = (1.0 - p.smoothing) * (fmax(-u, 0.0) + rest);
    if (p.smoothing > 0.0) loss += p.smoothing * (fmax(u, 0.0) + rest);  // (an infinite margin is no NaN)
    const double lesser = t / (1.0 + t), greater = 1.0 / (1.0 + t);  // sigmoid(-|u|), sigmoid(|u|)
    const double above = u >= 0.0 ? greater : lesser, below = u >= 0.0 ? lesser : greater;  // sigmoid(u), sigmoid(-u)
    const float slope = (float)in_range(-p.beta * p.scale * ((1.0 - p.smoothing) * below - p.smoothing * above));
    if (threadIdx.x == 0) {
        if (p.margin) p.margin[pair] = (float)u;
        p.pair_loss[pair] = (float)(p.scale * loss);
    }
    if (!p.grad) return;
    for (int64_t row = begin + half; row < end; row += 128)
        p.slope[row] = p.inverse[row] == 0.0f ? 0.0f : threadIdx.x >> 7 ? -slope : slope;
}

__global__ void k_set_float(float *to, float value) { *to = value; }

hipError_t launch_set_float(float *to, float value, hipStream_t stream) {
    k_set_float<<<1, 1, 0, stream>>>(to, value);
    return hipGetLastError();
}

#define OMK_BY_TYPE(type, CALL)     \
    switch (type) {                 \
        case OMK_F32: {             \
            typedef float T;        \
            CALL;                   \
        } break;                    \
        case OMK_BF16: {            \
            typedef bf16_t T;       \
            CALL;                   \
        } break;                    \
        default: {                  \
            typedef f16_t T;        \
            CALL;                   \
        }                           \
    }

int64_t wide_work(int64_t rows, int32_t actions) {
    // (rows of 32-bit logits are cut into twice the pieces: enough for either width)
    if (actions <= kMostInRegisters) return 0;
    const int64_t pieces = (actions + Pack<float>::V + piece_elements<float>() - 2) / piece_elements<float>();
    return rows * (pieces * (int64_t)sizeof(RowStats) + (int64_t)sizeof(Move)) + 16;
}

hipError_t launch_priors(int type, const Rows &r, float *priors, int64_t prior_stride, void *work, hipStream_t stream) {
    Launched l;
    OMK_BY_TYPE(type, l = type_priors<T>(r, priors, prior_stride, work, stream));
    return l.error;
}

hipError_t launch_logprobs(int type, const Rows &r, const int32_t *moves, float *logprob, float *entropy, void *work,
                           hipStream_t stream) {
    Launched l;
    OMK_BY_TYPE(type, l = type_logprobs<T>(r, moves, logprob, entropy, work, stream));
    return l.error;
}

hipError_t launch_policy_loss(int type, const Rows &r, const PolicyLoss &p, hipStream_t stream) {
    Launched l;
    OMK_BY_TYPE(type, l = type_policy_loss<T>(r, p, stream));
    if (l.error != hipSuccess || l.shares == 1) return l.error;
    k_sum<<<1, kSumBlock, 0, stream>>>(p.shares, l.shares, p.loss);
    return hipGetLastError();
}

hipError_t launch_preference_loss(int type, const Rows &r, const PreferenceLoss &p, int64_t before, hipStream_t stream) {
    hipError_t e = hipSuccess;
    if (!p.pairs) {  // rows of no line: the gradient's launch sets them, and the loss, to 0
        OMK_BY_TYPE(type, e = type_line_gradient<T>(r, p, stream));
        return e;
    }
    if (r.rows) {
        Launched l;
        OMK_BY_TYPE(type, l = type_lines<T>(r, p, before, stream));
        if (l.error != hipSuccess) return l.error;
    }
    k_pairs<<<(unsigned)p.pairs, 256, 0, stream>>>(r, p);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (p.grad) {
        OMK_BY_TYPE(type, e = type_line_gradient<T>(r, p, stream));
        return e;
    }
    k_sum<<<1, kSumBlock, 0, stream>>>(p.pair_loss, p.pairs, p.loss);
    return hipGetLastError();
}

}  // namespace omk
