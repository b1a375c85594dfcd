// Kernels over rows of logits.  What they all compute, per row: m = max over the legal x, S = sum exp(x - m); then an
// operator's few numbers per row, and from exp(x - m) its output per element.  k_rows reads every row once: a team of
// lanes holds it in registers from the look for its largest logit to the writing of its gradient (or priors).
// Rows too wide for that are cut into pieces (k_parts, k_apply) and read twice.
// Instantiated per type of the logits by omk_policy_{f32,bf16,f16}.hip.
#pragma once

#include "omk_learn_device.h"
#include "omk_learn_internal.h"

namespace omk {

// What a row (or a part of one) comes to: its largest legal logit (0 if there is none), the sum of exp(x - top) (x - top)
// over the legal ones, and the sum of exp(x - top) (0: no policy).
struct RowStats {
    float top, centred;
    double sum;
};

// ---- 16 bytes of a row ----

// Vectors of a row lie at multiples of 16 bytes of the matrix, not of the row: the first holds `head` elements of what
// lies before the row, so that rows of any width are read by whole vectors.  (Without `aligned`: rows are cut from
// their first element, and vectors are put together element by element.)
template <typename T>
__device__ __forceinline__ int head_of(const Rows &r, int64_t row) {
    return r.aligned ? (int)((uint64_t)(row * r.stride) & (Pack<T>::V - 1)) : 0;
}

// Bits of the elements j .. j + V - 1 that are the row's.
template <int V>
__device__ __forceinline__ uint32_t inside_bits(int j, int actions) {
    uint32_t b = (1u << V) - 1u;
    if (j < 0) b &= b << -j;
    if (j + V > actions) b = j < actions ? b & ((1u << (actions - j)) - 1u) : 0u;
    return b;
}

// Bits of the elements that are legal (of those that are the row's): from two neighbouring words at once.
__device__ __forceinline__ uint32_t legal_bits(const uint32_t *legal, int words, int j) {
    const int at = j < 0 ? 0 : j;
    uint32_t bits;
    if (words > 1) {
        struct __attribute__((packed, aligned(4))) Pair {
            uint64_t both;
        };
        const int w = min(at >> 5, words - 2);
        bits = (uint32_t)(((const Pair *)(legal + w))->both >> (at - 32 * w));
    } else {
        bits = legal[0] >> at;
    }
    return j < 0 ? bits << -j : bits;
}

// ONCE: the matrix is larger than the caches, and what is read or written now is not met again in them (nontemporal loads
// and stores).
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <bool ONCE>
__device__ __forceinline__ uint4 load16(const void *from) {
    if constexpr (ONCE) return __builtin_bit_cast(uint4, __builtin_nontemporal_load((const u32x4 *)from));
    return *(const uint4 *)from;
}
template <bool ONCE>
__device__ __forceinline__ void store16(void *to, uint4 v) {
    if constexpr (ONCE)
        __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), (u32x4 *)to);
    else
        *(uint4 *)to = v;
}

template <bool ONCE, typename T>
__device__ __forceinline__ void load_vector(const Rows &r, int64_t row, int j, uint32_t inside, Pack<T> &p) {
    constexpr int V = Pack<T>::V;
    const int64_t at = row * r.stride + j;
    if (!inside) return;
    if (r.aligned && at + V <= r.span) {  // (at >= 0: the matrix begins at a multiple of 16 bytes)
        p.raw = load16<ONCE>((const T *)r.x + at);
        return;
    }
#pragma unroll
    for (int i = 0; i < V; i++)
        if (inside >> i & 1u) p.x[i] = ((const T *)r.x)[at + i];
}

template <bool ONCE, typename T, typename OUT>
__device__ __forceinline__ void store_vector(OUT *out, bool aligned, int j, int actions, const float (&y)[Pack<T>::V]) {
    constexpr int V = Pack<T>::V;
    if (aligned && j >= 0 && j + V <= actions) {
        if constexpr (sizeof(OUT) == sizeof(T)) {
            Pack<OUT> p;
#pragma unroll
            for (int i = 0; i < V; i++) p.x[i] = (OUT)y[i];
            store16<ONCE>(out + j, p.raw);
        } else {  // 32-bit results of 16-bit logits
#pragma unroll
            for (int i = 0; i < V; i += 4)
                store16<ONCE>(out + j + i, __builtin_bit_cast(uint4, make_float4(y[i], y[i + 1], y[i + 2], y[i + 3])));
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < V; i++)
        if (j + i >= 0 && j + i < actions) out[j + i] = (OUT)y[i];
}

// ---- what operators do with a row ----

// The move of a row (-1 where it lies outside the action space) and its logit, -inf where it is not legal.
struct Move {
    int32_t move;
    float chosen;
};
template <typename T>
__device__ __forceinline__ Move move_of(const Rows &r, const int32_t *moves, int64_t row) {
    Move m = {moves ? moves[row] : -1, -INFINITY};
    if ((uint32_t)m.move >= (uint32_t)r.actions) m.move = -1;
    if (m.move >= 0 && (!r.legal || (r.legal[row * r.legal_stride + (m.move >> 5)] >> (m.move & 31) & 1u)))
        m.chosen = (float)((const T *)r.x)[row * r.stride + m.move];
    return m;
}

// The result of an operator's look at a row: element j becomes each * exp(x_j - top), and at_move where j is the move (a
// gradient's slope * (1 - p), by itself: as slope and slope * -p it would lose its digits where p is nearly 1); 0 wherever `none`.
struct RowOut {
    float each, at_move;
    int32_t move;
    bool none;
    double share;  // of the loss
};

struct PriorsOp {
    static constexpr bool kCentred = false, kElements = true, kMoves = false, kLoss = false;
    template <typename T>
    using Element = float;
    const int32_t *moves;  // nullptr
    double *block_loss;    // nullptr
    float *priors;
    int64_t stride;
    bool aligned;
    template <typename OUT>
    __device__ OUT *elements(int64_t row) const {
        return priors + row * stride;
    }
    __device__ bool skips(const Rows &, int64_t) const { return false; }
    __device__ RowOut row(int64_t, const RowStats &s, Move, bool) const {
        return {s.sum == 0.0 ? 0.0f : 1.0f / (float)s.sum, 0.0f, -1, s.sum == 0.0, 0.0f};
    }
};

struct LogprobsOp {
    static constexpr bool kCentred = true, kElements = false, kMoves = true, kLoss = false;
    const int32_t *moves;
    double *block_loss;  // nullptr
    float *logprob, *entropy;
    __device__ bool skips(const Rows &, int64_t) const { return false; }
    __device__ RowOut row(int64_t row, const RowStats &s, Move m, bool writes) const {
        if (writes) {
            const double log_sum = log(s.sum);
            if (entropy) entropy[row] = s.sum == 0.0 ? 0.0f : (float)(log_sum - (double)(s.centred / (float)s.sum));
            if (logprob)
                logprob[row] = m.move < 0       ? 0.0f
                               : s.sum == 0.0 ? -INFINITY
                                              : (float)((double)m.chosen - (double)s.top - log_sum);
        }
        return {0.0f, 0.0f, -1, true, 0.0f};
    }
};

// exp(d) - d - 1 and its derivative, exp(d) - 1, in 64 bits (a row's alone).  Near 0, where both cancel, the first by its series
// d^2/2 (1 + d/3 (1 + d/4 (1 + d/5))), whose next term is below 2^-44 of the sum for |d| < 2^-6, and the second as the first and d;
// elsewhere the difference to 1 loses 7 of 53 bits at most.  Far below 0 the derivative is -1, at d = -inf too, where the
// value is infinite: made from the value it would be what is left of two numbers of d's magnitude.
struct Divergence {
    double value, slope;
};
__device__ __forceinline__ Divergence divergence(double d) {
    const double slope = exp(d) - 1.0;
    if (!(fabs(d) < 0x1p-6)) return {slope - d, slope};
    const double value = 0.5 * d * d * (1.0 + d * (1.0 / 3.0) * (1.0 + d * (1.0 / 4.0) * (1.0 + d * (1.0 / 5.0))));
    return {value, d + value};
}

// A derivative by a log-probability, as a 32-bit number: held at the ends of their range, since times the probability 0 of an
// illegal action an infinite one would be no number.  (NaN stays.)
__device__ __forceinline__ double in_range(double slope) {
    const double most = 0x1.fffffep127;
    return slope > most ? most : slope < -most ? -most : slope;
}

// 1 / x for 1 <= x < 2^30: a 32-bit one, a step off, and Newton's step in 64 bits (good to 2^-44).
__device__ __forceinline__ double reciprocal(double x) {
    const double r = (double)__builtin_amdgcn_rcpf((float)x);
    return r * __builtin_fma(-x, r, 2.0);
}

struct PolicyOp {
    static constexpr bool kCentred = false, kElements = true, kMoves = true, kLoss = true;
    template <typename T>
    using Element = T;
    const int32_t *moves;
    double *block_loss;  // a block's share of the loss, by the block's number (by the row where rows are cut)
    PolicyLoss p;
    bool aligned;
    __device__ bool skips(const Rows &, int64_t) const { return false; }
    __device__ void add(int64_t block, double share) const {
        if (block_loss)
            block_loss[block] = share;
        else
            *p.loss = (float)share;
    }
    template <typename OUT>
    __device__ OUT *elements(int64_t row) const {
        return p.grad ? (OUT *)p.grad + row * p.grad_stride : nullptr;
    }
    __device__ RowOut row(int64_t row, const RowStats &s, Move m, bool writes) const {
        // (in 64 bits up to the sum: advantages have a mean of about 0, and what is left of a sum of rows is small beside them)
        double loss = 0.0, slope = 0.0, others = 0.0;  // (probability of the other actions)
        float lp = 0.0f, kl = 0.0f;
        if (m.chosen != -INFINITY) {
            const double exact = (double)m.chosen - (double)s.top - log(s.sum);
            lp = (float)exact;
            // (a move with more than half of the probability has the largest logit, whose term is 1 exactly: nothing is lost of S - 1;
            // and beside a smaller term's S - e its rounding is nothing.  An exponential in 64 bits took 0.8 us of 69 on 131072 rows of 362.)
            if (p.grad) others = (s.sum - (double)exp_of<true>(at_least(m.chosen - s.top, -200.0f))) * reciprocal(s.sum);
            const float a = p.advantage[row];
            const double shift = exact - (double)p.old_logprob[row];
            if (a > 0.0f ? shift > p.log_high : a < 0.0f && shift < p.log_low) {
                loss = -(a > 0.0f ? p.high : p.low) * (double)a;
            } else if (a != 0.0f) {
                loss = slope = -exp(shift) * (double)a;
            }
            if (p.ref_logprob) {
                const Divergence from = divergence((double)p.ref_logprob[row] - exact);
                kl = (float)from.value;
                if (p.kl_weight > 0.0) {  // (a divergence that is only reported may be infinite)
                    loss += p.kl_weight * from.value;
                    slope -= p.kl_weight * from.slope;
                }
            }
            const double w = (p.weight ? (double)p.weight[row] : 1.0) * p.scale;
            loss = w == 0.0 ? 0.0 : loss * w;
            slope = w == 0.0 ? 0.0 : slope * w;
        }
        if (writes) {
            p.logprob[row] = lp;
            if (p.kl) p.kl[row] = kl;
        }
        slope = in_range(slope);
        const float by_logprob = (float)slope;
        return {by_logprob == 0.0f ? 0.0f : -by_logprob * __builtin_amdgcn_rcpf((float)s.sum),
                by_logprob == 0.0f ? 0.0f : (float)(slope * others), m.move, by_logprob == 0.0f, loss};
    }
};

// The rows that lines hold: from line_begin's first to its last, inside the rows there are.  (None without pairs, where
// line_begin may be NULL.)
struct LineRows {
    int64_t begin, end;
    __device__ int64_t inside(int64_t at) const { return at < begin ? begin : at > end ? end : at; }
};
__device__ __forceinline__ LineRows line_rows(const PreferenceLoss &p, int64_t rows) {
    if (p.pairs == 0) return {0, 0};
    const LineRows all = {0, rows};
    const int64_t begin = all.inside(p.line_begin[0]), end = all.inside(p.line_begin[2 * p.pairs]);
    return {begin, end < begin ? begin : end};
}

struct LineOp {
    static constexpr bool kCentred = false, kElements = false, kMoves = true, kLoss = false;
    const int32_t *moves;
    double *block_loss;  // nullptr
    PreferenceLoss p;
    __device__ bool skips(const Rows &r, int64_t row) const {
        const LineRows lines = line_rows(p, r.rows);
        return row < lines.begin || row >= lines.end;
    }
    __device__ RowOut row(int64_t row, const RowStats &s, Move m, bool writes) const {
        if (writes) {
            const bool counts = m.chosen != -INFINITY;
            p.top[row] = s.top;
            p.inverse[row] = counts ? 1.0f / (float)s.sum : 0.0f;
            p.logprob[row] = counts ? (double)m.chosen - (double)s.top - log(s.sum) : 0.0;
            p.slope[row] = 0.0f;  // until its line says otherwise
        }
        return {0.0f, 0.0f, -1, true, 0.0f};
    }
};

// ---- rows that registers hold ----

// sum exp(x - m) (x - m) of terms relative to their own maximum m, relative to one that is -d larger: f is exp(d).  (d is bounded
// as single terms' differences are below: where f is 0 long since, a sum of terms at the type's lowest value times d would
// be infinite, and the product no number.)
__device__ __forceinline__ float moved(float centred, float sum, float d, float f) {
    return (centred + sum * fmaxf(d, -200.0f)) * f;
}

// Joins the maxima and sums of a block's wavefronts, whose terms are relative to their own maxima until then: one
// exchange through LDS serves both.  Every thread of the block calls it; the result is the same in all of them.  A lane for
// every wavefront, so that its factor can be taken in 64 bits: in 32 its rounding would be in all of the wavefront's terms alike.
template <bool CENTRED, int WAVES>
__device__ __forceinline__ RowStats join_waves(float top, double sum, float centred) {
    __shared__ float tops[WAVES], centreds[WAVES];
    __shared__ double sums[WAVES];
    const int wave = threadIdx.x >> 6, of = threadIdx.x & (WAVES - 1);
    if ((threadIdx.x & 63) == 0) {
        tops[wave] = top;
        sums[wave] = sum;
        if (CENTRED) centreds[wave] = centred;
    }
    __syncthreads();
    const float its = tops[of];
    RowStats all = {team_max<WAVES>(its), 0.0f, 0.0};
    if (all.top == -INFINITY) all.top = 0.0f;
    const double d = its == -INFINITY ? 0.0 : (double)its - (double)all.top, f = exp(d);  // (an empty one's sum is 0, or NaN)
    all.sum = team_sum<WAVES>(sums[of] * f);
    if (CENTRED) all.centred = team_sum<WAVES>(moved(centreds[of], (float)sums[of], (float)d, (float)f));
    return all;
}

// exp(x - m) of a vector's elements; with CENTRED also adds exp(x - m) (x - m) up, where a term whose exponential is 0 (x = -inf
// among them) counts nothing and one that is no number shows.
template <bool FINE, bool CENTRED, int V>
__device__ __forceinline__ void exponentials(const float (&x)[V], float top, float (&e)[V], float &centred) {
#pragma unroll
    for (int i = 0; i < V; i++) {
        const float d = FINE ? at_least(x[i] - top, -200.0f) : x[i] - top;
        e[i] = exp_of<FINE>(d);
        if (CENTRED) centred = __builtin_fmaf(e[i], d, centred);
    }
}

// Their sum.  In 64 bits from the terms on: beside the largest, which is 1, the others of a row that is all but decided would lose
// their digits, and with them the logarithm of the sum.
template <int V>
__device__ __forceinline__ double sum_of(const float (&e)[V]) {
    double even = (double)e[0], odd = (double)e[1];
#pragma unroll
    for (int i = 2; i < V; i += 2) {
        even += (double)e[i];
        odd += (double)e[i + 1];
    }
    return even + odd;
}

// The elements of a vector as floats, -inf where they are not the row's or not legal.  LOOK: nearly all vectors of a row
// without a mask are whole in every lane, and need no look at single elements.  (Not where registers are short: two
// ways through the code keep more alive.)
template <bool LOOK, typename T>
__device__ __forceinline__ void floats_of(const Pack<T> &p, uint32_t bits, float (&x)[Pack<T>::V]) {
    constexpr int V = Pack<T>::V;
    if (LOOK && __all(bits == (1u << V) - 1u)) {
#pragma unroll
        for (int i = 0; i < V; i++) x[i] = (float)p.x[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) {
            // (the bit spread over a word, and the value or -inf picked by it: two instructions)
            const uint32_t all = (uint32_t)((int32_t)(bits << (31 - i)) >> 31);
            x[i] = __uint_as_float((__float_as_uint((float)p.x[i]) & all) | (0xFF800000u & ~all));
        }
    }
}

// Writes a vector of a row's results: exp(x - m) times `each`, but `at_move` at element `at` (counted from the first
// vector's first; -1: nowhere), or 0.
template <bool ONCE, typename T, typename OUT>
__device__ __forceinline__ void write_vector(OUT *to, bool aligned, int vec, int head, int actions, const float (&e)[Pack<T>::V],
                                             float each, bool none, int at, float at_move) {
    constexpr int V = Pack<T>::V;
    float y[V];
#pragma unroll
    for (int i = 0; i < V; i++) y[i] = none ? 0.0f : e[i] * each;
    if (at >= 0 && at / V == vec) {
#pragma unroll
        for (int i = 0; i < V; i++) y[i] = at % V == i ? at_move : y[i];
    }
    store_vector<ONCE, T, OUT>(to, aligned, vec * V - head, actions, y);
}

// Narrow rows: TEAM lanes (of a wavefront's 64) hold a row, K vectors a lane.  What bounds it is the instructions, of which
// elements are the smaller part: the reductions and a row's few numbers (its log-probability, the loss and its
// slope: some 300) cost the same for a row in 8 lanes as for one in 64, and are shared by all rows of the wavefront.
template <bool ONCE, typename T, int TEAM, int K, typename OP>
__global__ __launch_bounds__(256) void k_narrow(Rows r, OP op) {
    constexpr int V = Pack<T>::V;
    const int sub = threadIdx.x & (TEAM - 1);
    const int64_t row = r.first + (int64_t)blockIdx.x * (256 / TEAM) + threadIdx.x / TEAM;
    const bool here = row < r.rows && !op.skips(r, row);
    const int head = here ? head_of<T>(r, row) : 0;
    // (loaded before this wavefront, which alone writes these rows' gradients, writes any: they may lie where the logits are)
    Move m = {-1, -INFINITY};
    if (OP::kMoves && here && sub == 0) m = move_of<T>(r, op.moves, row);
    Pack<T> p[K];
    uint32_t bits[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int j = (k * TEAM + sub) * V - head;
        bits[k] = here ? inside_bits<V>(j, r.actions) : 0u;
        load_vector<ONCE, T>(r, row, j, bits[k], p[k]);
    }
    if (r.legal) {
#pragma unroll
        for (int k = 0; k < K; k++)
            if (bits[k]) bits[k] &= legal_bits(r.legal + row * r.legal_stride, r.words, (k * TEAM + sub) * V - head);
    }
    float e[K][V], top = -INFINITY;
#pragma unroll
    for (int k = 0; k < K; k++) {
        floats_of<true, T>(p[k], bits[k], e[k]);
#pragma unroll
        for (int i = 0; i < V; i++) top = fmaxf(top, e[k][i]);
    }
    top = team_max<TEAM>(top);
    if (top == -INFINITY) top = 0.0f;
    double sum = 0.0;
    float centred = 0.0f;
#pragma unroll
    for (int k = 0; k < K; k++) {
        exponentials<true, OP::kCentred, V>(e[k], top, e[k], centred);
        sum += sum_of<V>(e[k]);
    }
    if (OP::kCentred) centred = team_sum<TEAM>(centred);
    const RowStats s = {top, centred, team_sum<TEAM>(sum)};
    RowOut out = {0.0f, 0.0f, -1, true, 0.0f};
    if (here && sub == 0) out = op.row(row, s, m, true);

    if constexpr (OP::kElements) {
        typedef typename OP::template Element<T> OUT;
        if (op.template elements<OUT>(0)) {
            const float each = __shfl(out.each, 0, TEAM), at_move = __shfl(out.at_move, 0, TEAM);
            const int move = __shfl(out.move, 0, TEAM);
            const bool none = __shfl((int)out.none, 0, TEAM);
            OUT *to = op.template elements<OUT>(row);
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int vec = k * TEAM + sub;
                if (here && vec * V - head < r.actions)
                    write_vector<ONCE, T, OUT>(to, op.aligned, vec, head, r.actions, e[k], each, none,
                                               move < 0 ? -1 : move + head, at_move);
            }
        }
    }
    if constexpr (OP::kLoss) {
        __shared__ double shares[4];
        const double share = team_sum<64>(out.share);
        if ((threadIdx.x & 63) == 0) shares[threadIdx.x >> 6] = share;
        __syncthreads();
        if (threadIdx.x == 0) op.add(blockIdx.x, shares[0] + shares[1] + (shares[2] + shares[3]));
    }
}

// Wider rows: a block of TEAM threads holds a row, K vectors a thread.
//
// What bounds it is memory's rate, if enough loads are on their way: a block that waits for its row's reductions loads
// nothing, so a compute unit needs two of the largest blocks (at most 64 registers a thread; with one at a time these rows took
// half as much again).  8192 rows of 32768 bf16 with their gradient take 206 to 212 us one call behind another (5.1 to 5.2 TB/s).
template <bool ONCE, typename T, int TEAM, int K, typename OP>
__global__ __launch_bounds__(TEAM, TEAM == 1024 && K <= 4 ? 8 : 1) void k_rows(Rows r, OP op) {
    constexpr int V = Pack<T>::V, WAVES = TEAM / 64;
    // exp(x - m) stays in registers, up to 32 of them; wider rows compute it again from the logits
    constexpr bool KEEP = K * V <= 32;
    const int64_t row = r.first + blockIdx.x;
    if (op.skips(r, row)) return;
    const int head = head_of<T>(r, row);

    // (the wavefront that looks at the move writes no other's part of the row before it has used what it found: the
    // gradient may lie where the logits are)
    Move m = {-1, -INFINITY};
    if (OP::kMoves && threadIdx.x < 64) m = move_of<T>(r, op.moves, row);
    Pack<T> p[K];
    uint32_t bits[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int j = (k * TEAM + (int)threadIdx.x) * V - head;
        bits[k] = inside_bits<V>(j, r.actions);
        load_vector<ONCE, T>(r, row, j, bits[k], p[k]);
    }
    if (r.legal) {
        const uint32_t *legal = r.legal + row * r.legal_stride;
#pragma unroll
        for (int k = 0; k < K; k++)
            if (bits[k]) bits[k] &= legal_bits(legal, r.words, (k * TEAM + (int)threadIdx.x) * V - head);
    }
    float e[KEEP ? K : 1][V];
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < K; k++) {
        float(&x)[V] = e[KEEP ? k : 0];
        floats_of<false, T>(p[k], bits[k], x);
#pragma unroll
        for (int i = 0; i < V; i++) top = fmaxf(top, x[i]);
    }
    top = team_max<64>(top);
    const float own_top = top == -INFINITY ? 0.0f : top;
    double sum = 0.0;
    float centred = 0.0f;
#pragma unroll
    for (int k = 0; k < K; k++) {
        float(&x)[V] = e[KEEP ? k : 0];
        if (!KEEP) floats_of<false, T>(p[k], bits[k], x);
        exponentials<true, OP::kCentred, V>(x, own_top, x, centred);
        sum += sum_of<V>(x);
    }
    if (OP::kCentred) centred = team_sum<64>(centred);
    __shared__ RowOut shared_out;
    const RowStats s = join_waves<OP::kCentred, WAVES>(top, team_sum<64>(sum), centred);
    if (threadIdx.x < 64) {
        const RowOut o = op.row(row, s, m, threadIdx.x == 0);
        if (threadIdx.x == 0) shared_out = o;
    }
    if constexpr (OP::kElements) {
        __syncthreads();
        typedef typename OP::template Element<T> OUT;
        const RowOut out = shared_out;
        if (OUT *to = op.template elements<OUT>(row)) {
            const float each = out.each * (top == -INFINITY ? 0.0f : exp_of<true>(at_least(top - s.top, -200.0f)));
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int vec = k * TEAM + (int)threadIdx.x;
                float(&x)[V] = e[KEEP ? k : 0];
                if (!KEEP) {
                    floats_of<false, T>(p[k], bits[k], x);
                    exponentials<false, false, V>(x, own_top, x, centred);
                }
                if (vec * V - head < r.actions)
                    write_vector<ONCE, T, OUT>(to, op.aligned, vec, head, r.actions, x, each, out.none,
                                               out.move < 0 ? -1 : out.move + head, out.at_move);
            }
        }
    }
    if constexpr (OP::kLoss)
        if (threadIdx.x == 0) op.add(blockIdx.x, shared_out.share);
}

// ---- rows of which nothing but numbers is wanted ----

constexpr int kTile = 2;  // vectors of a thread at a time

// A block goes through vectors first .. end - 1 of a row tile by tile with a running maximum and sum: m' = max(m, tile's
// maximum), s' = s exp(m - m') + sum exp(x - m').  The next tile is on its way while one is looked at, and few registers hold
// it all, so that eight blocks share a compute unit.  (Tiles of four vectors were slower by a tenth: five blocks.)  2049 rows of 50001
// f16 with their entropies: 56 us, 3.7 TB/s, bound by instructions: 15 a term, four of them the exponential's.
template <bool ONCE, typename T, int BLOCK, bool CENTRED>
__device__ __forceinline__ RowStats stream_row(const Rows &r, int64_t row, int first, int end) {
    constexpr int V = Pack<T>::V;
    const int head = head_of<T>(r, row);
    const uint32_t *legal = r.legal ? r.legal + row * r.legal_stride : nullptr;
    Pack<T> next[kTile];
    const auto bits_at = [&](int vec) { return vec < end ? inside_bits<V>(vec * V - head, r.actions) : 0u; };
    // Tiles that lie inside the row are loaded without a look at bounds, and without a mask need none at bits either (the rows
    // above: 64 us where every tile looks, 56 us so).
    const T *const at_row = (const T *)r.x + (row * r.stride - head);
    const int inner_end = min(end, (r.actions + head) / V);
    const auto inner = [&](int start) { return r.aligned && (start || !head) && start + kTile * BLOCK <= inner_end; };
    const auto load = [&](int start) {
        const int from = start + (int)threadIdx.x;
        if (inner(start)) {
#pragma unroll
            for (int k = 0; k < kTile; k++) next[k].raw = load16<ONCE>(at_row + (from + k * BLOCK) * V);
            return;
        }
#pragma unroll
        for (int k = 0; k < kTile; k++)
            load_vector<ONCE, T>(r, row, (from + k * BLOCK) * V - head, bits_at(from + k * BLOCK), next[k]);
    };
    load(first);
    float top = -INFINITY, centred = 0.0f;
    double sum = 0.0;
    for (int start = first; start < end; start += kTile * BLOCK) {
        const int from = start + (int)threadIdx.x;
        float x[kTile][V], most = top;
        const bool all = !legal && inner(start);
#pragma unroll
        for (int k = 0; k < kTile; k++) {
            uint32_t bits = (1u << V) - 1u;
            if (!all) {
                bits = bits_at(from + k * BLOCK);
                if (legal && bits) bits &= legal_bits(legal, r.words, (from + k * BLOCK) * V - head);
            }
            floats_of<true, T>(next[k], bits, x[k]);
#pragma unroll
            for (int i = 0; i < V; i++) most = fmaxf(most, x[k][i]);
        }
        load(start + kTile * BLOCK);
        const float at = most == -INFINITY ? 0.0f : most, d = at_least(top - at, -200.0f), f = exp_of<true>(d);
        if (CENTRED) centred = top == -INFINITY ? 0.0f : moved(centred, (float)sum, d, f);
        sum *= (double)f;
#pragma unroll
        for (int k = 0; k < kTile; k++) {
            exponentials<true, CENTRED, V>(x[k], at, x[k], centred);
            sum += sum_of<V>(x[k]);
        }
        top = most;
    }
    // the lanes' maxima and sums, then the wavefronts'
    const float most = team_max<64>(top);
    const double d = top == -INFINITY ? 0.0 : (double)top - (double)most, f = exp(d);
    if (CENTRED) centred = team_sum<64>(moved(centred, (float)sum, (float)d, (float)f));
    return join_waves<CENTRED, BLOCK / 64>(most, team_sum<64>(sum * f), centred);
}

template <bool ONCE, typename T, int BLOCK, typename OP>
__global__ __launch_bounds__(BLOCK) void k_stream(Rows r, OP op) {
    const int64_t row = r.first + blockIdx.x;
    if (op.skips(r, row)) return;
    const int vectors = (r.actions + head_of<T>(r, row) + Pack<T>::V - 1) / Pack<T>::V;
    Move m = {-1, -INFINITY};
    if (threadIdx.x < 64) m = move_of<T>(r, op.moves, row);
    const RowStats s = stream_row<ONCE, T, BLOCK, OP::kCentred>(r, row, 0, vectors);
    if (threadIdx.x < 64) op.row(row, s, m, threadIdx.x == 0);
}

// ---- rows cut into pieces ----

constexpr int kPieceBlock = 256;
constexpr int kPieceVectors = 8;  // of a thread

template <typename T>
__host__ __device__ constexpr int piece_elements() {
    return kPieceBlock * kPieceVectors * Pack<T>::V;
}

struct Wide {
    int32_t pieces;
    RowStats *parts;  // [rows][pieces]
    Move *moves;      // [rows]: looked up before any gradient is written where logits may be
};

template <bool ONCE, typename T, typename OP>
__global__ __launch_bounds__(kPieceBlock) void k_parts(Rows r, OP op, Wide w) {
    const int64_t row = blockIdx.x / w.pieces;
    if (op.skips(r, row)) return;
    const int piece = blockIdx.x % w.pieces, first = piece * (kPieceVectors * kPieceBlock);
    RowStats s = stream_row<ONCE, T, kPieceBlock, OP::kCentred>(r, row, first, first + kPieceVectors * kPieceBlock);
    if (threadIdx.x) return;
    if (s.sum == 0.0) s.top = -INFINITY;  // nothing here: no maximum for the row's
    w.parts[blockIdx.x] = s;
    if (OP::kMoves && piece == 0) w.moves[row] = move_of<T>(r, op.moves, row);
}

// A block for every piece (for every row where an operator has no elements).
template <bool ONCE, typename T, typename OP>
__global__ __launch_bounds__(kPieceBlock) void k_apply(Rows r, OP op, Wide w) {
    constexpr int V = Pack<T>::V, K = kPieceVectors;
    const int64_t row = OP::kElements ? blockIdx.x / w.pieces : blockIdx.x;
    if (op.skips(r, row)) return;
    const int piece = OP::kElements ? blockIdx.x % w.pieces : 0;
    const RowStats *parts = w.parts + row * w.pieces;
    // a thread's parts, then its wavefront's, then the block's
    float top = -INFINITY;
    for (int i = threadIdx.x; i < w.pieces; i += kPieceBlock) top = fmaxf(top, parts[i].top);
    top = team_max<64>(top);
    double sum = 0.0;
    float centred = 0.0f;
    for (int i = threadIdx.x; i < w.pieces; i += kPieceBlock) {
        const bool empty = parts[i].top == -INFINITY;
        const double d = empty ? 0.0 : (double)parts[i].top - (double)top, f = exp(d);
        sum += parts[i].sum * f;
        if (OP::kCentred) centred += moved(parts[i].centred, (float)parts[i].sum, (float)d, (float)f);
    }
    if (OP::kCentred) centred = team_sum<64>(centred);
    const RowStats s = join_waves<OP::kCentred, kPieceBlock / 64>(top, team_sum<64>(sum), centred);
    __shared__ RowOut shared_out;
    if (threadIdx.x < 64) {
        const Move m = OP::kMoves ? w.moves[row] : Move{-1, -INFINITY};
        const RowOut o = op.row(row, s, m, piece == 0 && threadIdx.x == 0);
        if (threadIdx.x == 0) {
            shared_out = o;
            if constexpr (OP::kLoss)
                if (piece == 0) op.add(row, o.share);
        }
    }
    if constexpr (OP::kElements) {
        __syncthreads();
        typedef typename OP::template Element<T> OUT;
        const RowOut out = shared_out;
        OUT *to = op.template elements<OUT>(row);
        if (!to) return;
        const int head = head_of<T>(r, row), first = piece * (K * kPieceBlock) + threadIdx.x;
        const int at = out.move < 0 ? -1 : out.move + head;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int vec = first + k * kPieceBlock, j = vec * V - head;
            if (j >= r.actions) continue;
            Pack<T> p;
            uint32_t bits = inside_bits<V>(j, r.actions);
            load_vector<ONCE, T>(r, row, j, bits, p);
            if (r.legal) bits &= legal_bits(r.legal + row * r.legal_stride, r.words, j);
            float x[V], unused = 0.0f;
            floats_of<true, T>(p, bits, x);
            exponentials<false, false, V>(x, s.top, x, unused);
            write_vector<ONCE, T, OUT>(to, op.aligned, vec, head, r.actions, x, out.each, out.none, at, out.at_move);
        }
    }
}

// ---- the gradient of rows whose slope is known ----

constexpr int kGradientVectors = 4;  // of a lane

// The sum of n values by one block, in one order whatever runs beside it: in its first thread.
template <int BLOCK, typename F>
__device__ __forceinline__ double block_sum(const F *values, int64_t n) {
    __shared__ double part[BLOCK / 64];
    double s = 0.0;
    // (eight at a time, so that as many loads are on their way)
    int64_t i = threadIdx.x;
    for (; i + 7 * BLOCK < n; i += 8 * BLOCK) {
        F v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = values[i + k * BLOCK];
#pragma unroll
        for (int k = 0; k < 8; k++) s += (double)v[k];
    }
    for (; i < n; i += BLOCK) s += (double)values[i];
    s = team_sum<64>(s);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0.0;
    for (int w = 0; w < BLOCK / 64; w++) s += part[w];
    return s;
}

// The gradient's slope is known only when the last row of a pair has been read, so that logits are read twice: 9728 rows of
// 32768 bf16 (638 MB) in 335 us, of which the first reading takes 122 us (5.2 TB/s) and this, which reads again and writes, 211 us
// (6.0 TB/s).
// Two and eight vectors a lane took a fifth longer than four.
// A wavefront takes kGradientVectors * 64 vectors of a row.  The first block also adds the pairs' losses up.
// Rows are taken from the last to the first: those that the
// look at all rows has read last are in the cache still.
template <bool ONCE, typename T>
__global__ __launch_bounds__(256) void k_line_gradient(Rows r, PreferenceLoss p, bool aligned, int pieces, int64_t first_block) {
    constexpr int V = Pack<T>::V, K = kGradientVectors;
    const int lane = threadIdx.x & 63;
    if (first_block + blockIdx.x == 0) {
        const double loss = block_sum<256>(p.pair_loss, p.pairs);
        if (threadIdx.x == 0) *p.loss = (float)loss;
    }
    const int64_t item = (first_block + blockIdx.x) * 4 + (threadIdx.x >> 6), back = item / pieces;
    if (back >= r.rows) return;
    const int64_t row = r.rows - 1 - back;
    const LineRows lines = line_rows(p, r.rows);
    const bool rest = row < lines.begin || row >= lines.end;
    if (rest && !p.zero_rest) return;
    const float slope = rest ? 0.0f : p.slope[row], top = rest ? 0.0f : p.top[row];
    const float each = rest ? 0.0f : -slope * p.inverse[row];
    const int piece = (int)(item % pieces), head = head_of<T>(r, row), first = piece * (K * 64) + lane;
    const int at = slope == 0.0f ? -1 : p.moves[row] + head;
    float at_move = 0.0f;
    if (at >= 0 && at / (V * K * 64) == piece) at_move = (float)((double)slope * (1.0 - exp(p.logprob[row])));
    T *to = (T *)p.grad + row * p.grad_stride;
    Pack<T> x[K];
    uint32_t bits[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int j = (first + k * 64) * V - head;
        bits[k] = slope == 0.0f ? 0u : inside_bits<V>(j, r.actions);
        load_vector<ONCE, T>(r, row, j, bits[k], x[k]);
    }
    if (r.legal) {
#pragma unroll
        for (int k = 0; k < K; k++)
            if (bits[k]) bits[k] &= legal_bits(r.legal + row * r.legal_stride, r.words, (first + k * 64) * V - head);
    }
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int vec = first + k * 64, j = vec * V - head;
        if (j >= r.actions) continue;
        float e[V], unused = 0.0f;
        floats_of<true, T>(x[k], bits[k], e);
        exponentials<false, false, V>(e, top, e, unused);
        write_vector<ONCE, T, T>(to, aligned, vec, head, r.actions, e, each, slope == 0.0f, at, at_move);
    }
}

// ---- which kernel ----

// Vectors of the widest row, whatever its head.
template <typename T>
static inline int64_t vectors_of(const Rows &r) {
    constexpr int V = Pack<T>::V;
    const int64_t most = r.actions + (r.aligned && r.rows > 1 && r.stride % V ? V - 1 : 0);
    return (most + V - 1) / V;
}

// Blocks of a launch, which leave a share of the loss each (rows, where they are cut).  A single one writes the loss itself.
struct Launched {
    hipError_t error;
    int64_t shares;
};

// A launch's threads are counted in 32 bits: 2^21 blocks (of 1024 at most) at a time.
constexpr int64_t kMostBlocks = 1 << 21;

template <typename OP, typename LAUNCH>
static Launched launch_rows(const Rows &r, const OP &op, int64_t per_block, const LAUNCH &launch) {
    const int64_t blocks = (r.rows + per_block - 1) / per_block;
    Rows some = r;
    OP o = op;
    if constexpr (OP::kLoss)
        if (blocks == 1) o.block_loss = nullptr;  // its share is the loss
    hipError_t e = hipSuccess;
    for (int64_t b = 0; b < blocks && e == hipSuccess; b += kMostBlocks) {
        some.first = b * per_block;
        launch(some, o, (unsigned)(blocks - b < kMostBlocks ? blocks - b : kMostBlocks));
        e = hipGetLastError();
        if constexpr (OP::kLoss)
            if (o.block_loss) o.block_loss += kMostBlocks;
    }
    return {e, blocks};
}

template <bool ONCE, typename T, int TEAM, int K, typename OP>
static Launched run_narrow(const Rows &r, const OP &op, hipStream_t stream) {
    return launch_rows(r, op, 256 / TEAM, [&](const Rows &some, const OP &o, unsigned blocks) {
        k_narrow<ONCE, T, TEAM, K, OP><<<blocks, 256, 0, stream>>>(some, o);
    });
}

template <bool ONCE, typename T, int TEAM, int K, typename OP>
static Launched run_rows(const Rows &r, const OP &op, hipStream_t stream) {
    return launch_rows(r, op, 1, [&](const Rows &some, const OP &o, unsigned blocks) {
        k_rows<ONCE, T, TEAM, K, OP><<<blocks, TEAM, 0, stream>>>(some, o);
    });
}

template <bool ONCE, typename T, int BLOCK, typename OP>
static Launched run_stream(const Rows &r, const OP &op, hipStream_t stream) {
    return launch_rows(r, op, 1, [&](const Rows &some, const OP &o, unsigned blocks) {
        k_stream<ONCE, T, BLOCK, OP><<<blocks, BLOCK, 0, stream>>>(some, o);
    });
}

// Wavefronts that fill the card: eight on each of 256 compute units.  (Rows of 362 bf16 with their gradient: 4096 of them
// take 8.0 us with 64 lanes each and 8.9 us with 16, 8192 12.7 and 9.7 us, 16384 21.3 and 15.0 us, 131072 130 and 71 us.)
constexpr int64_t kFullOfRows = 256 * 8;

template <bool ONCE, typename T, typename OP>
static Launched run_class(const Rows &r, const OP &op, const Wide &w, hipStream_t stream) {
    const int64_t n = vectors_of<T>(r);
    // Few rows are done soonest with a lane for every vector; where the card is full of wavefronts all the same, many
    // rows to a wavefront: four vectors a lane and 16 lanes at least (with 8 a store's pieces are shorter than a cache
    // line: 131072 rows of 225 floats took a fifth longer than with 16).
    if (n <= 256) {
        const auto full = [&](int team) { return r.rows >= kFullOfRows * (64 / team); };
        if (n <= 32 && full(16)) return run_narrow<ONCE, T, 16, 2>(r, op, stream);
        if (n <= 32) return run_narrow<ONCE, T, 32, 1>(r, op, stream);
        if (n <= 64 && full(16)) return run_narrow<ONCE, T, 16, 4>(r, op, stream);
        if (n <= 64) return run_narrow<ONCE, T, 64, 1>(r, op, stream);
        if (n <= 128 && full(32)) return run_narrow<ONCE, T, 32, 4>(r, op, stream);
        if (n <= 128) return run_narrow<ONCE, T, 64, 2>(r, op, stream);
        return run_narrow<ONCE, T, 64, 4>(r, op, stream);
    }
    if (n <= 512) return run_rows<ONCE, T, 256, 2>(r, op, stream);
    if constexpr (OP::kElements) {
        if (n <= 1024) return run_rows<ONCE, T, 256, 4>(r, op, stream);
        if (n <= 2048) return run_rows<ONCE, T, 1024, 2>(r, op, stream);
        if (n <= 4096) return run_rows<ONCE, T, 1024, 4>(r, op, stream);
        if (n <= 8192) return run_rows<ONCE, T, 1024, 8>(r, op, stream);
        if constexpr (sizeof(T) == 4)
            if (n <= 16384) return run_rows<ONCE, T, 1024, 16>(r, op, stream);
    } else if (n <= 16384) {
        // (up to a row for every compute unit: 64 rows of 32768 bf16 take 6.9 us with blocks of 1024 and 9.0 us with blocks of 256,
        // 256 rows 7.6 and 9.5 us, 384 rows 13.3 and 12.8 us, 512 rows 14.0 and 13.2 us, 1024 rows 21.1 and 18.6 us)
        return r.rows <= 256 ? run_stream<ONCE, T, 1024>(r, op, stream) : run_stream<ONCE, T, 256>(r, op, stream);
    }
    OP o = op;
    if constexpr (OP::kLoss)
        if (r.rows == 1) o.block_loss = nullptr;  // its share is the loss
    k_parts<ONCE, T, OP><<<(unsigned)(r.rows * w.pieces), kPieceBlock, 0, stream>>>(r, o, w);
    k_apply<ONCE, T, OP><<<(unsigned)(OP::kElements ? r.rows * w.pieces : r.rows), kPieceBlock, 0, stream>>>(r, o, w);
    return {hipGetLastError(), r.rows};
}

// Logits that the second-level caches (4 MB on each of the card's eight dies) cannot hold together are not kept in them:
// 8192 rows of 32768 bf16 take 221 us with nontemporal accesses and 233 us without, 131072 of 362 (95 MB) 70 and 76 us,
// 32768 of 362 floats (47 MB) 29.4 and 28.1 us.
static inline bool met_once(const Rows &r, int width) { return r.rows * (int64_t)r.actions * width > (int64_t)32 << 20; }

template <typename T, typename OP>
static Launched run(const Rows &r, const OP &op, const Wide &w, hipStream_t stream) {
    return met_once(r, sizeof(T)) ? run_class<true, T>(r, op, w, stream) : run_class<false, T>(r, op, w, stream);
}

// Work space of rows that are cut into pieces, at the end of what the caller gives (behind `before` bytes).
template <typename T>
static Wide wide_of(const Rows &r, void *work, int64_t before) {
    Wide w = {(int32_t)((vectors_of<T>(r) + kPieceBlock * kPieceVectors - 1) / (kPieceBlock * kPieceVectors)), nullptr, nullptr};
    w.parts = (RowStats *)((char *)work + (before + 15) / 16 * 16);
    w.moves = (Move *)(w.parts + r.rows * w.pieces);
    return w;
}

// Bases at multiples of 16 bytes and strides that agree in the vectors' lengths: then results have the logits' heads.
template <typename T>
static bool aligned_with(const Rows &r, const void *d, int64_t stride) {
    return r.aligned && ((uintptr_t)d & 15) == 0 && (r.rows < 2 || (stride - r.stride) % Pack<T>::V == 0);
}

template <typename T>
Launched type_priors(const Rows &r, float *priors, int64_t stride, void *work, hipStream_t stream) {
    const PriorsOp op = {nullptr, nullptr, priors, stride, aligned_with<T>(r, priors, stride)};
    return run<T>(r, op, wide_of<T>(r, work, 0), stream);
}

template <typename T>
Launched type_logprobs(const Rows &r, const int32_t *moves, float *logprob, float *entropy, void *work, hipStream_t stream) {
    const LogprobsOp op = {logprob ? moves : nullptr, nullptr, logprob, entropy};
    return run<T>(r, op, wide_of<T>(r, work, 0), stream);
}

template <typename T>
Launched type_policy_loss(const Rows &r, const PolicyLoss &p, hipStream_t stream) {
    const PolicyOp op = {p.moves, p.shares, p, p.grad && aligned_with<T>(r, p.grad, p.grad_stride)};
    return run<T>(r, op, wide_of<T>(r, p.shares, r.rows * 8), stream);
}

template <typename T>
Launched type_lines(const Rows &r, const PreferenceLoss &p, int64_t before, hipStream_t stream) {
    const LineOp op = {p.moves, nullptr, p};
    return run<T>(r, op, wide_of<T>(r, p.work, before), stream);
}

template <typename T>
hipError_t type_line_gradient(const Rows &r, const PreferenceLoss &p, hipStream_t stream) {
    const int64_t pieces = (vectors_of<T>(r) + 64 * kGradientVectors - 1) / (64 * kGradientVectors);
    const int64_t blocks = (r.rows * pieces + 3) / 4;
    const bool aligned = aligned_with<T>(r, p.grad, p.grad_stride);
    hipError_t e = hipSuccess;
    for (int64_t b = 0; b < blocks && e == hipSuccess; b += kMostBlocks) {
        const dim3 grid((unsigned)(blocks - b < kMostBlocks ? blocks - b : kMostBlocks));
        if (met_once(r, sizeof(T)))
            k_line_gradient<true, T><<<grid, 256, 0, stream>>>(r, p, aligned, (int)pieces, b);
        else
            k_line_gradient<false, T><<<grid, 256, 0, stream>>>(r, p, aligned, (int)pieces, b);
        e = hipGetLastError();
    }
    return e;
}

#define OMK_POLICY_TYPE(WORD, T)                                                                                         \
    WORD template Launched type_priors<T>(const Rows &, float *, int64_t, void *, hipStream_t);                          \
    WORD template Launched type_logprobs<T>(const Rows &, const int32_t *, float *, float *, void *, hipStream_t);       \
    WORD template Launched type_policy_loss<T>(const Rows &, const PolicyLoss &, hipStream_t);                           \
    WORD template Launched type_lines<T>(const Rows &, const PreferenceLoss &, int64_t, hipStream_t);                    \
    WORD template hipError_t type_line_gradient<T>(const Rows &, const PreferenceLoss &, hipStream_t);

}  // namespace omk
