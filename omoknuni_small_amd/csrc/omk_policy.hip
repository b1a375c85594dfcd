// Rows of logits: priors and log-probabilities of moves, the clipped policy loss and the preference loss with their
// gradients (include/omk_learn.h).
#include "omk_learn_device.h"
#include "omk_learn_internal.h"

namespace omk {

constexpr int kRowBlock = 256;  // threads: a wavefront takes a row
constexpr int kRowsPerBlock = kRowBlock / 64;

__device__ __forceinline__ bool is_legal(const uint32_t *legal, int j) { return !legal || (legal[j >> 5] >> (j & 31) & 1u); }

template <typename T>
struct OneRow {
    const T *x;
    const uint32_t *legal;
    __device__ OneRow(const Rows &r, int64_t row)
        : x((const T *)r.x + row * r.stride), legal(r.legal ? r.legal + row * r.legal_stride : nullptr) {}
    // -inf where the action is not legal
    __device__ float at(int j) const { return is_legal(legal, j) ? (float)x[j] : -INFINITY; }
};

template <bool CENTRED, typename T>
__device__ RowStats row_stats(const OneRow<T> &row, int actions, int lane) {
    float top = -INFINITY;
    for (int j = lane; j < actions; j += 64) top = fmaxf(top, row.at(j));
    top = wave_max(top);
    RowStats s = {top > -INFINITY ? top : 0.0f, 0.0f, 0.0f};
    for (int j = lane; j < actions; j += 64) {
        const float d = row.at(j) - s.top, e = exp_of(d);
        s.sum += e;
        if (CENTRED && e > 0.0f) s.centred += e * d;
    }
    s.sum = wave_sum(s.sum);
    if (CENTRED) s.centred = wave_sum(s.centred);
    return s;
}

template <typename T>
__global__ __launch_bounds__(kRowBlock) void k_priors(Rows r, float *priors, int64_t prior_stride) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * kRowsPerBlock + (threadIdx.x >> 6);
    if (row >= r.rows) return;
    const OneRow<T> x(r, row);
    const RowStats s = row_stats<false>(x, r.actions, lane);
    const float inverse = s.sum == 0.0f ? 0.0f : 1.0f / s.sum;
    for (int j = lane; j < r.actions; j += 64) priors[row * prior_stride + j] = exp_of(x.at(j) - s.top) * inverse;
}

template <typename T>
__global__ __launch_bounds__(kRowBlock) void k_logprobs(Rows r, const int32_t *moves, float *logprob, float *entropy) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * kRowsPerBlock + (threadIdx.x >> 6);
    if (row >= r.rows) return;
    const OneRow<T> x(r, row);
    const RowStats s = row_stats<true>(x, r.actions, lane);
    if (lane) return;
    const double log_sum = log_of_sum(s.sum);
    if (entropy) entropy[row] = s.sum == 0.0f ? 0.0f : (float)(log_sum - (double)(s.centred / s.sum));
    if (logprob) {
        const int move = moves[row];
        float lp = 0.0f;
        if ((uint32_t)move < (uint32_t)r.actions)
            lp = s.sum == 0.0f ? -INFINITY : (float)((double)x.at(move) - (double)s.top - log_sum);
        logprob[row] = lp;
    }
}

// The row's share of the loss and its derivative by the move's log-probability, both before weight and scale.
struct RowLoss {
    float loss, slope, kl;
};

// exp(d) - d - 1 without the cancellation near 0: d^2/2 (1 + d/3 (1 + d/4 (..))), whose first term left out is below
// 2^-24 of the sum for |d| < 1/4
__device__ __forceinline__ float exp_minus_linear(float d, float expm1_d) {
    if (fabsf(d) >= 0.25f) return expm1_d - d;
    float s = 1.0f + d * (1.0f / 9.0f);
    s = 1.0f + d * (1.0f / 8.0f) * s;
    s = 1.0f + d * (1.0f / 7.0f) * s;
    s = 1.0f + d * (1.0f / 6.0f) * s;
    s = 1.0f + d * (1.0f / 5.0f) * s;
    s = 1.0f + d * (1.0f / 4.0f) * s;
    s = 1.0f + d * (1.0f / 3.0f) * s;
    return 0.5f * d * d * s;
}

__device__ __forceinline__ RowLoss clipped_loss(const PolicyLoss &p, double lp, int64_t row) {
    const float a = p.advantage[row];
    const double shift = lp - (double)p.old_logprob[row];
    RowLoss o = {0.0f, 0.0f, 0.0f};
    if (a > 0.0f ? shift > p.log_high : a < 0.0f && shift < p.log_low) {
        o.loss = -(a > 0.0f ? p.high : p.low) * a;
    } else if (a != 0.0f) {
        o.loss = o.slope = -expf((float)shift) * a;
    }
    if (p.ref_logprob) {
        const float d = (float)((double)p.ref_logprob[row] - lp), e = expm1f(d);
        o.kl = exp_minus_linear(d, e);
        o.loss += p.kl_weight * o.kl;
        o.slope -= p.kl_weight * e;
    }
    return o;
}

template <typename T>
__device__ void write_gradient(const OneRow<T> &x, int actions, const RowStats &s, int move, float slope, T *grad, int lane) {
    const float each = slope == 0.0f ? 0.0f : -slope * (1.0f / s.sum);
    for (int j = lane; j < actions; j += 64) {
        float g = 0.0f;
        if (slope != 0.0f) g = exp_of(x.at(j) - s.top) * each + (j == move ? slope : 0.0f);
        grad[j] = (T)g;
    }
}

template <typename T>
__global__ __launch_bounds__(kRowBlock) void k_policy_loss(Rows r, PolicyLoss p) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * kRowsPerBlock + (threadIdx.x >> 6);
    if (row >= r.rows) return;
    const OneRow<T> x(r, row);
    const int move = p.moves[row];
    const bool inside = (uint32_t)move < (uint32_t)r.actions;
    const float chosen = inside ? x.at(move) : -INFINITY;
    RowStats s = {0.0f, 1.0f, 0.0f};
    RowLoss l = {0.0f, 0.0f, 0.0f};
    float lp = 0.0f, w = 0.0f;
    if (chosen != -INFINITY) {
        s = row_stats<false>(x, r.actions, lane);
        const double exact = (double)chosen - (double)s.top - log_of_sum(s.sum);
        lp = (float)exact;
        l = clipped_loss(p, exact, row);
        w = (p.weight ? p.weight[row] : 1.0f) * p.scale;
    }
    if (lane == 0) {
        p.logprob[row] = lp;
        if (p.kl) p.kl[row] = l.kl;
        p.row_loss[row] = chosen != -INFINITY ? w * l.loss : 0.0f;
    }
    if (p.grad)
        write_gradient(x, r.actions, s, move, chosen != -INFINITY ? w * l.slope : 0.0f, (T *)p.grad + row * p.grad_stride,
                       lane);
}

constexpr int kSumBlock = 1024;

// The sum of n values, in one order whatever runs beside it.
__global__ __launch_bounds__(kSumBlock) void k_sum(const float *values, int64_t n, float *out) {
    __shared__ double part[kSumBlock / 64];
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += kSumBlock) s += (double)values[i];
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x) return;
    s = 0.0;
    for (int i = 0; i < kSumBlock / 64; i++) s += part[i];
    *out = (float)s;
}

// ---- preference loss: the rows' log-probabilities, then every pair's loss, then the rows' gradients ----

// The rows that lines hold: line_begin's first to its last, inside the rows there are.
struct LineRows {
    int64_t begin, end;
};
__device__ __forceinline__ int64_t inside(int64_t at, int64_t rows) { return at < 0 ? 0 : at > rows ? rows : at; }
__device__ __forceinline__ LineRows line_rows(const PreferenceLoss &p, int64_t rows) {
    return {inside(p.line_begin[0], rows), inside(p.line_begin[2 * p.pairs], rows)};
}

template <typename T>
__global__ __launch_bounds__(kRowBlock) void k_line_rows(Rows r, PreferenceLoss p) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * kRowsPerBlock + (threadIdx.x >> 6);
    const LineRows lines = line_rows(p, r.rows);
    if (row < lines.begin || row >= lines.end) return;
    const OneRow<T> x(r, row);
    const int move = p.moves[row];
    const float chosen = (uint32_t)move < (uint32_t)r.actions ? x.at(move) : -INFINITY;
    RowStats s = {0.0f, 0.0f, 0.0f};
    float lp = 0.0f;
    if (chosen != -INFINITY) {
        s = row_stats<false>(x, r.actions, lane);
        lp = (float)((double)chosen - (double)s.top - log_of_sum(s.sum));
    }
    if (lane == 0) {
        p.top[row] = s.top;
        p.inverse[row] = chosen != -INFINITY ? 1.0f / s.sum : 0.0f;
        p.logprob[row] = lp;
        p.slope[row] = 0.0f;  // until its line says otherwise
    }
}

// A wavefront for every pair.
__global__ __launch_bounds__(kRowBlock) void k_pairs(Rows r, PreferenceLoss p) {
    const int lane = threadIdx.x & 63;
    const int64_t pair = (int64_t)blockIdx.x * kRowsPerBlock + (threadIdx.x >> 6);
    if (pair >= p.pairs) return;
    double sums[2];
    for (int side = 0; side < 2; side++) {
        const int64_t line = 2 * pair + side;
        const int64_t begin = inside(p.line_begin[line], r.rows), end = inside(p.line_begin[line + 1], r.rows);
        double s = 0.0;
        for (int64_t row = begin + lane; row < end; row += 64) s += (double)p.logprob[row];
        sums[side] = wave_sum(s);
        if (lane == 0 && p.line_logprob) p.line_logprob[line] = (float)sums[side];
        if (p.ref_logprob) sums[side] -= (double)p.ref_logprob[line];
    }
    const float u = (float)((double)p.beta * (sums[0] - sums[1]));
    // log(1 + exp(-|u|)), of which both losses are made
    const float t = expf(-fabsf(u)), rest = log1pf(t);
    float loss = (1.0f - p.smoothing) * (fmaxf(-u, 0.0f) + rest);
    if (p.smoothing > 0.0f) loss += p.smoothing * (fmaxf(u, 0.0f) + rest);  // (an infinite margin is no NaN)
    const float lesser = t / (1.0f + t), greater = 1.0f / (1.0f + t);  // sigmoid(-|u|), sigmoid(|u|)
    const float above = u >= 0.0f ? greater : lesser, below = u >= 0.0f ? lesser : greater;  // sigmoid(u), sigmoid(-u)
    const float slope = -p.beta * p.scale * ((1.0f - p.smoothing) * below - p.smoothing * above);
    if (lane == 0) {
        if (p.margin) p.margin[pair] = u;
        p.pair_loss[pair] = p.scale * loss;
    }
    if (!p.grad) return;
    for (int side = 0; side < 2; side++) {
        const int64_t line = 2 * pair + side;
        const int64_t begin = inside(p.line_begin[line], r.rows), end = inside(p.line_begin[line + 1], r.rows);
        for (int64_t row = begin + lane; row < end; row += 64)
            p.slope[row] = p.inverse[row] == 0.0f ? 0.0f : side ? -slope : slope;
    }
}

template <typename T>
__global__ __launch_bounds__(kRowBlock) void k_line_gradient(Rows r, PreferenceLoss p) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * kRowsPerBlock + (threadIdx.x >> 6);
    const LineRows lines = line_rows(p, r.rows);
    const bool rest = row < lines.begin || row >= lines.end;
    if (row >= r.rows || (rest && !p.zero_rest)) return;
    const OneRow<T> x(r, row);
    const RowStats s = {rest ? 0.0f : p.top[row], rest ? 1.0f : 1.0f / p.inverse[row], 0.0f};
    write_gradient(x, r.actions, s, p.moves[row], rest ? 0.0f : p.slope[row], (T *)p.grad + row * p.grad_stride, lane);
}

__global__ void k_set_float(float *to, float value) { *to = value; }

hipError_t launch_set_float(float *to, float value, hipStream_t stream) {
    k_set_float<<<1, 1, 0, stream>>>(to, value);
    return hipGetLastError();
}

static inline dim3 row_grid(int64_t rows) { return dim3((unsigned)((rows + kRowsPerBlock - 1) / kRowsPerBlock)); }

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

hipError_t launch_priors(int type, const Rows &r, float *priors, int64_t prior_stride, hipStream_t stream) {
    OMK_BY_TYPE(type, (k_priors<T><<<row_grid(r.rows), kRowBlock, 0, stream>>>(r, priors, prior_stride)));
    return hipGetLastError();
}

hipError_t launch_logprobs(int type, const Rows &r, const int32_t *moves, float *logprob, float *entropy,
                           hipStream_t stream) {
    OMK_BY_TYPE(type, (k_logprobs<T><<<row_grid(r.rows), kRowBlock, 0, stream>>>(r, moves, logprob, entropy)));
    return hipGetLastError();
}

hipError_t launch_policy_loss(int type, const Rows &r, const PolicyLoss &p, hipStream_t stream) {
    OMK_BY_TYPE(type, (k_policy_loss<T><<<row_grid(r.rows), kRowBlock, 0, stream>>>(r, p)));
    k_sum<<<1, kSumBlock, 0, stream>>>(p.row_loss, r.rows, p.loss);
    return hipGetLastError();
}

hipError_t launch_preference_loss(int type, const Rows &r, const PreferenceLoss &p, hipStream_t stream) {
    if (r.rows) OMK_BY_TYPE(type, (k_line_rows<T><<<row_grid(r.rows), kRowBlock, 0, stream>>>(r, p)));
    k_pairs<<<row_grid(p.pairs), kRowBlock, 0, stream>>>(r, p);
    k_sum<<<1, kSumBlock, 0, stream>>>(p.pair_loss, p.pairs, p.loss);
    if (p.grad) OMK_BY_TYPE(type, (k_line_gradient<T><<<row_grid(r.rows), kRowBlock, 0, stream>>>(r, p)));
    return hipGetLastError();
}

}  // namespace omk
