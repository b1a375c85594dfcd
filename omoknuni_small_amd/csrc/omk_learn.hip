// C ABI of include/omk_learn.h: handles, checks of arguments, and the launches.
#include "../../include/omk_learn.h"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <exception>
#include <initializer_list>
#include <new>
#include <utility>
#include <vector>

#include "omk_learn_internal.h"

using namespace omk;

struct omk_learner {
    int device = 0;
    hipStream_t stream = nullptr;
    int children = 0;       // optimizers that live
    bool released = false;  // omk_learner_destroy was called while some did
};

struct omk_adamw {
    omk_learner *l = nullptr;
    int32_t n_tensors = 0;
    int32_t param_type = 0, grad_type = 0, copy_type = 0, state_type = 0;
    double beta1 = 0, beta2 = 0, eps = 0;
    uint32_t seed = 0;
    int32_t chunk_units = 0;
    char *memory = nullptr;  // the count and its groups' counters, the tensors, the chunks
    uint32_t *done = nullptr;
    AdamCount *count = nullptr;
    AdamTensor *tensors = nullptr;
    AdamChunk *chunks = nullptr;
    std::vector<int64_t> first_chunk;  // of every tensor, and the end
    std::vector<int64_t> elements;
};

namespace {

// The calling thread's device is the learner's while one of these lives.
struct OnDevice {
    int before = -1;
    hipError_t status;
    explicit OnDevice(int device) {
        status = hipGetDevice(&before);
        if (status == hipSuccess && before != device) status = hipSetDevice(device);
        if (status == hipSuccess && before == device) before = -1;
        (void)hipGetLastError();  // launches are checked with hipGetLastError: start from a clean slate
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

#define LEARN_TRY(expr)                                                                                \
    do {                                                                                               \
        hipError_t e_ = (expr);                                                                        \
        if (e_ != hipSuccess) return learn_fail(OMK_ERR_HIP, "%s: %s", #expr, hipGetErrorString(e_)); \
    } while (0)

// No C++ exception crosses the C boundary.
#define LEARN_NO_THROW \
    catch (const std::exception &e_) { return learn_fail(OMK_ERR_INVALID, "out of host memory (%s)", e_.what()); }

int width_of(int type) { return type == OMK_F32 ? 4 : type == OMK_F8 ? 1 : 2; }
bool float_type(int type) { return type == OMK_F32 || type == OMK_BF16 || type == OMK_F16; }
bool aligned(const void *p, int width) { return ((uintptr_t)p & (uintptr_t)(width - 1)) == 0; }

// Bytes from the first element of a matrix to behind its last; -1 where that passes 2^46, which no address space holds.
int64_t span_bytes(int64_t rows, int64_t stride, int64_t columns, int width) {
    const __int128 n = ((__int128)(rows - 1) * stride + columns) * width;
    return n >> 46 ? -1 : (int64_t)n;
}

bool overlap(const void *a, int64_t a_bytes, const void *b, int64_t b_bytes) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + (uintptr_t)b_bytes && y < x + (uintptr_t)a_bytes;
}

int check_rows(const char *who, const omk_policy_rows *r, Rows *out) {
    if (!float_type(r->type)) return learn_fail(OMK_ERR_INVALID, "%s: logits of type %d", who, r->type);
    if (r->rows < 0 || r->rows > INT32_MAX)
        return learn_fail(OMK_ERR_INVALID, "%s: %lld rows", who, (long long)r->rows);
    if (r->actions < 1 || r->actions > OMK_MAX_ACTIONS)
        return learn_fail(OMK_ERR_INVALID, "%s: %d actions (1 .. %d)", who, r->actions, OMK_MAX_ACTIONS);
    const int words = (r->actions + 31) / 32;
    if (r->rows > 1 && r->row_stride < r->actions)
        return learn_fail(OMK_ERR_INVALID, "%s: rows of %d actions, %lld apart", who, r->actions, (long long)r->row_stride);
    if (r->d_legal && (r->legal_stride < 0 || (r->rows > 1 && r->legal_stride && r->legal_stride < words)))
        return learn_fail(OMK_ERR_INVALID, "%s: masks of %d words, %lld apart", who, words, (long long)r->legal_stride);
    if (r->rows && !r->d_logits) return learn_fail(OMK_ERR_INVALID, "%s: no logits", who);
    if (!aligned(r->d_logits, width_of(r->type)) || !aligned(r->d_legal, 4))
        return learn_fail(OMK_ERR_INVALID, "%s: an address that is no multiple of its type's size", who);
    if (r->rows && (span_bytes(r->rows, r->row_stride, r->actions, width_of(r->type)) < 0 ||
                    (r->d_legal && span_bytes(r->rows, r->legal_stride, words, 4) < 0)))
        return learn_fail(OMK_ERR_INVALID, "%s: rows that pass the address space", who);
    *out = Rows{r->d_logits, r->row_stride, r->rows, r->actions, 0, r->d_legal, r->legal_stride, words,
                r->rows ? (r->rows - 1) * r->row_stride + r->actions : 0, aligned(r->d_logits, 16)};
    return OMK_OK;
}

// A matrix of results beside the logits: apart from them, or (in_place) just where they are.
int check_result(const char *who, const char *what, const omk_policy_rows *r, const void *d, int64_t stride, int width,
                 bool in_place) {
    if (!d) return learn_fail(OMK_ERR_INVALID, "%s: no %s", who, what);
    if (!aligned(d, width)) return learn_fail(OMK_ERR_INVALID, "%s: %s at an address that is no multiple of its type's size", who, what);
    if (r->rows > 1 && stride < r->actions)
        return learn_fail(OMK_ERR_INVALID, "%s: %s rows of %d actions, %lld apart", who, what, r->actions, (long long)stride);
    const int64_t bytes = span_bytes(r->rows, stride, r->actions, width);
    if (bytes < 0) return learn_fail(OMK_ERR_INVALID, "%s: rows that pass the address space", who);
    const int64_t of_logits = span_bytes(r->rows, r->row_stride, r->actions, width_of(r->type));
    if (in_place && d == r->d_logits && (r->rows < 2 || stride == r->row_stride)) return OMK_OK;
    if (overlap(d, bytes, r->d_logits, of_logits))
        return learn_fail(OMK_ERR_INVALID, "%s: the %s lies across the logits", who, what);
    return OMK_OK;
}

int check_work(const char *who, const void *d_work, int64_t work_bytes, int64_t needed) {
    if (!aligned(d_work, 16)) return learn_fail(OMK_ERR_INVALID, "%s: work space at an address that is no multiple of 16", who);
    if (needed && (!d_work || work_bytes < needed))
        return learn_fail(OMK_ERR_CAPACITY, "%s: %lld bytes of work space, %lld needed", who,
                          (long long)(d_work ? work_bytes : 0), (long long)needed);
    return OMK_OK;
}

// Bytes of memory, or of every row of a matrix.
struct Piece {
    const void *at;
    int64_t bytes, stride = 0, rows = 1;
};

bool across(const Piece &a, const Piece &b) {
    if (!a.at || !b.at || !a.bytes || !b.bytes) return false;
    if (a.rows > 1 && b.rows > 1)  // (two matrices: what lies between rows counts)
        return overlap(a.at, (a.rows - 1) * a.stride + a.bytes, b.at, (b.rows - 1) * b.stride + b.bytes);
    if (a.rows > 1) return across(b, a);
    // the first of b's rows that ends behind a's beginning
    const int64_t from = (int64_t)((uintptr_t)a.at - (uintptr_t)b.at);
    const int64_t row = from < b.bytes || b.rows < 2 ? 0 : (from - b.bytes) / b.stride + 1;
    return row < b.rows && overlap(a.at, a.bytes, (const char *)b.at + row * b.stride, b.bytes);
}

Piece logits_of(const omk_policy_rows *r) {
    const int width = width_of(r->type);
    return {r->d_logits, (int64_t)r->actions * width, r->row_stride * width, r->rows};
}
Piece legal_of(const omk_policy_rows *r) {
    return {r->d_legal, (int64_t)((r->actions + 31) / 32) * 4, r->legal_stride * 4, r->legal_stride ? r->rows : 1};
}
// A matrix of results beside the logits.
Piece matrix_of(const omk_policy_rows *r, const void *d, int64_t stride, int width) {
    return {d, (int64_t)r->actions * width, stride * width, r->rows};
}

// Results, work space among them, lie apart from each other and from all that is read.  (The first is a matrix, which
// check_result has held against the logits, the first of what is read.)
int check_apart(const char *who, std::initializer_list<Piece> results, std::initializer_list<Piece> reads) {
    for (const Piece *a = results.begin(); a != results.end(); a++) {
        for (const Piece *b = reads.begin() + (a == results.begin()); b != reads.end(); b++)
            if (across(*a, *b)) return learn_fail(OMK_ERR_INVALID, "%s: a result lies across what is read", who);
        for (const Piece *b = a + 1; b != results.end(); b++)
            if (across(*a, *b)) return learn_fail(OMK_ERR_INVALID, "%s: two results lie across each other", who);
    }
    return OMK_OK;
}

bool aligned4(const char *who, const void *const *p, int n) {
    for (int i = 0; i < n; i++)
        if (!aligned(p[i], 4)) {
            learn_fail(OMK_ERR_INVALID, "%s: an address that is no multiple of its type's size", who);
            return false;
        }
    return true;
}

}  // namespace

extern "C" {

int omk_learner_create(int32_t device, omk_learner **out) {
    if (!out) return learn_fail(OMK_ERR_INVALID, "omk_learner_create: null argument");
    int count = 0;
    LEARN_TRY(hipGetDeviceCount(&count));
    if (device < 0 || device >= count)
        return learn_fail(OMK_ERR_INVALID, "omk_learner_create: device %d of %d", device, count);
    omk_learner *l = new (std::nothrow) omk_learner();
    if (!l) return learn_fail(OMK_ERR_INVALID, "out of host memory");
    l->device = device;
    *out = l;
    return OMK_OK;
}

int omk_learner_destroy(omk_learner *l) {
    if (l && l->children)
        l->released = true;  // goes with the last of its optimizers
    else
        delete l;
    return OMK_OK;
}

int omk_learner_set_stream(omk_learner *l, void *hip_stream) {
    if (!l) return learn_fail(OMK_ERR_INVALID, "omk_learner_set_stream: null argument");
    l->stream = (hipStream_t)hip_stream;
    return OMK_OK;
}

int omk_learner_get_stream(omk_learner *l, void **hip_stream_out) {
    if (!l || !hip_stream_out) return learn_fail(OMK_ERR_INVALID, "omk_learner_get_stream: null argument");
    *hip_stream_out = (void *)l->stream;
    return OMK_OK;
}

int omk_learner_sync(omk_learner *l) {
    if (!l) return learn_fail(OMK_ERR_INVALID, "omk_learner_sync: null argument");
    OnDevice on(l->device);
    LEARN_TRY(on.status);
    LEARN_TRY(hipStreamSynchronize(l->stream));
    return OMK_OK;
}

int64_t omk_policy_work(int64_t rows, int32_t actions) { return rows > 0 ? wide_work(rows, actions) : 0; }

int omk_policy_priors(omk_learner *l, const omk_policy_rows *rows, float *d_priors, int64_t prior_stride, void *d_work,
                      int64_t work_bytes) {
    const char *who = "omk_policy_priors";
    if (!l || !rows) return learn_fail(OMK_ERR_INVALID, "%s: null argument", who);
    Rows r;
    if (int rc = check_rows(who, rows, &r)) return rc;
    if (!r.rows) return OMK_OK;
    if (int rc = check_result(who, "priors", rows, d_priors, prior_stride, 4, false)) return rc;
    const int64_t work = omk_policy_work(r.rows, r.actions);
    if (int rc = check_work(who, d_work, work_bytes, work)) return rc;
    if (int rc = check_apart(who, {matrix_of(rows, d_priors, prior_stride, 4), {d_work, work}}, {logits_of(rows), legal_of(rows)}))
        return rc;
    OnDevice on(l->device);
    LEARN_TRY(on.status);
    LEARN_TRY(launch_priors(rows->type, r, d_priors, prior_stride, d_work, l->stream));
    return OMK_OK;
}

int omk_policy_logprobs(omk_learner *l, const omk_policy_rows *rows, const int32_t *d_moves, float *d_logprob,
                        float *d_entropy, void *d_work, int64_t work_bytes) {
    const char *who = "omk_policy_logprobs";
    if (!l || !rows) return learn_fail(OMK_ERR_INVALID, "%s: null argument", who);
    Rows r;
    if (int rc = check_rows(who, rows, &r)) return rc;
    if (d_logprob && !d_moves && r.rows) return learn_fail(OMK_ERR_INVALID, "%s: no moves", who);
    const void *all[] = {d_moves, d_logprob, d_entropy};
    if (!aligned4(who, all, 3)) return OMK_ERR_INVALID;
    if (!r.rows || (!d_logprob && !d_entropy)) return OMK_OK;
    const int64_t work = omk_policy_work(r.rows, r.actions), column = r.rows * 4;
    if (int rc = check_work(who, d_work, work_bytes, work)) return rc;
    if (int rc = check_apart(who, {{nullptr, 0}, {d_logprob, column}, {d_entropy, column}, {d_work, work}},
                             {logits_of(rows), legal_of(rows), {d_logprob ? d_moves : nullptr, column}}))
        return rc;
    OnDevice on(l->device);
    LEARN_TRY(on.status);
    LEARN_TRY(launch_logprobs(rows->type, r, d_moves, d_logprob, d_entropy, d_work, l->stream));
    return OMK_OK;
}

int64_t omk_policy_loss_work(int64_t rows, int32_t actions) {
    return rows > 0 ? (rows * 8 + 15) / 16 * 16 + wide_work(rows, actions) : 0;
}

int omk_policy_loss(omk_learner *l, const omk_policy_rows *rows, const omk_policy_samples *samples,
                    const omk_policy_loss_params *params, const omk_policy_loss_out *out, void *d_work,
                    int64_t work_bytes) {
    const char *who = "omk_policy_loss";
    if (!l || !rows || !samples || !params || !out) return learn_fail(OMK_ERR_INVALID, "%s: null argument", who);
    Rows r;
    if (int rc = check_rows(who, rows, &r)) return rc;
    if (!(params->clip_low >= 0.0) || !(params->clip_high >= 0.0) || !std::isfinite(params->clip_high))
        return learn_fail(OMK_ERR_INVALID, "%s: clipped to [1 - %g, 1 + %g]", who, params->clip_low, params->clip_high);
    if (!(params->kl_weight >= 0.0) || !std::isfinite(params->kl_weight) || !std::isfinite(params->scale))
        return learn_fail(OMK_ERR_INVALID, "%s: kl_weight %g, scale %g", who, params->kl_weight, params->scale);
    if (params->kl_weight > 0.0 && !samples->d_ref_logprob)
        return learn_fail(OMK_ERR_INVALID, "%s: a KL term needs the reference's log-probabilities", who);
    if (!out->d_loss) return learn_fail(OMK_ERR_INVALID, "%s: no loss", who);
    const void *all[] = {samples->d_moves, samples->d_old_logprob, samples->d_advantage, samples->d_ref_logprob,
                         samples->d_weight, out->d_loss, out->d_logprob, out->d_kl};
    if (!aligned4(who, all, 8)) return OMK_ERR_INVALID;
    if (r.rows) {
        if (!samples->d_moves || !samples->d_old_logprob || !samples->d_advantage || !out->d_logprob)
            return learn_fail(OMK_ERR_INVALID, "%s: null argument", who);
        if (out->d_grad)
            if (int rc = check_result(who, "gradient", rows, out->d_grad, out->grad_stride, width_of(rows->type), true))
                return rc;
        const int64_t work = omk_policy_loss_work(r.rows, r.actions), column = r.rows * 4;
        if (int rc = check_work(who, d_work, work_bytes, work)) return rc;
        if (int rc = check_apart(who,
                                 {matrix_of(rows, out->d_grad, out->grad_stride, width_of(rows->type)), {out->d_loss, 4},
                                  {out->d_logprob, column}, {out->d_kl, column}, {d_work, work}},
                                 {logits_of(rows), legal_of(rows), {samples->d_moves, column}, {samples->d_old_logprob, column},
                                  {samples->d_advantage, column}, {samples->d_ref_logprob, column}, {samples->d_weight, column}}))
            return rc;
    }
    OnDevice on(l->device);
    LEARN_TRY(on.status);
    if (!r.rows) {
        LEARN_TRY(launch_set_float(out->d_loss, 0.0f, l->stream));
        return OMK_OK;
    }
    PolicyLoss p;
    p.moves = samples->d_moves;
    p.old_logprob = samples->d_old_logprob;
    p.advantage = samples->d_advantage;
    p.ref_logprob = samples->d_ref_logprob;
    p.weight = samples->d_weight;
    p.log_low = params->clip_low < 1.0 ? std::log(1.0 - params->clip_low) : -INFINITY;
    p.log_high = std::log(1.0 + params->clip_high);
    p.low = 1.0 - params->clip_low;
    p.high = 1.0 + params->clip_high;
    p.kl_weight = params->kl_weight;
    p.scale = params->scale;
    p.grad = out->d_grad;
    p.grad_stride = out->grad_stride;
    p.logprob = out->d_logprob;
    p.kl = out->d_kl;
    p.shares = (double *)d_work;
    p.loss = out->d_loss;
    LEARN_TRY(launch_policy_loss(rows->type, r, p, l->stream));
    return OMK_OK;
}

// 20 bytes a row and 4 a pair
static int64_t preference_before(int64_t rows, int64_t pairs) {
    return ((rows > 0 ? rows * 20 : 0) + (pairs > 0 ? pairs * 4 : 0) + 15) / 16 * 16;
}

int64_t omk_preference_loss_work(int64_t rows, int32_t actions, int64_t pairs) {
    return preference_before(rows, pairs) + (rows > 0 ? wide_work(rows, actions) : 0);
}

int omk_preference_loss(omk_learner *l, const omk_policy_rows *rows, const int32_t *d_moves,
                        const int32_t *d_line_begin, int64_t pairs, const float *d_ref_logprob,
                        const omk_preference_params *params, const omk_preference_out *out, void *d_work,
                        int64_t work_bytes) {
    const char *who = "omk_preference_loss";
    if (!l || !rows || !params || !out) return learn_fail(OMK_ERR_INVALID, "%s: null argument", who);
    Rows r;
    if (int rc = check_rows(who, rows, &r)) return rc;
    if (pairs < 0 || pairs > OMK_MAX_PAIRS) return learn_fail(OMK_ERR_INVALID, "%s: %lld pairs", who, (long long)pairs);
    if (!std::isfinite(params->beta) || !std::isfinite(params->scale) || !(params->label_smoothing >= 0.0) ||
        !(params->label_smoothing <= 0.5))
        return learn_fail(OMK_ERR_INVALID, "%s: beta %g, label_smoothing %g (0 .. 0.5), scale %g", who, params->beta,
                          params->label_smoothing, params->scale);
    if (!out->d_loss) return learn_fail(OMK_ERR_INVALID, "%s: no loss", who);
    const void *all[] = {d_moves, d_line_begin, d_ref_logprob, out->d_loss, out->d_margin, out->d_line_logprob};
    if (!aligned4(who, all, 6)) return OMK_ERR_INVALID;
    if (r.rows && out->d_grad)
        if (int rc = check_result(who, "gradient", rows, out->d_grad, out->grad_stride, width_of(rows->type), true)) return rc;
    if (pairs) {
        if (!d_line_begin || (r.rows && !d_moves)) return learn_fail(OMK_ERR_INVALID, "%s: null argument", who);
        const int64_t work = omk_preference_loss_work(r.rows, r.actions, pairs);
        if (int rc = check_work(who, d_work, work_bytes, work)) return rc;
        const bool some = r.rows > 0;
        if (int rc = check_apart(who,
                                 {matrix_of(rows, some ? out->d_grad : nullptr, out->grad_stride, width_of(rows->type)),
                                  {out->d_loss, 4}, {out->d_margin, pairs * 4}, {out->d_line_logprob, pairs * 8}, {d_work, work}},
                                 {some ? logits_of(rows) : Piece{nullptr, 0}, some ? legal_of(rows) : Piece{nullptr, 0},
                                  {d_moves, r.rows * 4}, {d_line_begin, pairs * 8 + 4}, {d_ref_logprob, pairs * 8}}))
            return rc;
    } else if (r.rows) {
        if (int rc = check_apart(who, {matrix_of(rows, out->d_grad, out->grad_stride, width_of(rows->type)), {out->d_loss, 4}},
                                 {logits_of(rows)}))
            return rc;
    }
    OnDevice on(l->device);
    LEARN_TRY(on.status);
    if (!pairs && !(r.rows && out->d_grad && out->zero_rest)) {
        LEARN_TRY(launch_set_float(out->d_loss, 0.0f, l->stream));
        return OMK_OK;
    }
    PreferenceLoss p;
    p.moves = d_moves;
    p.line_begin = d_line_begin;
    p.pairs = pairs;
    p.ref_logprob = d_ref_logprob;
    p.beta = params->beta;
    p.smoothing = params->label_smoothing;
    p.scale = params->scale;
    p.grad = r.rows ? out->d_grad : nullptr;
    p.grad_stride = out->grad_stride;
    p.zero_rest = out->zero_rest;
    p.margin = out->d_margin;
    p.line_logprob = out->d_line_logprob;
    p.loss = out->d_loss;
    p.work = d_work;
    p.logprob = (double *)d_work;
    p.top = (float *)(p.logprob + r.rows);
    p.inverse = p.top + r.rows;
    p.slope = p.inverse + r.rows;
    p.pair_loss = p.slope + r.rows;
    LEARN_TRY(launch_preference_loss(rows->type, r, p, preference_before(r.rows, pairs), l->stream));
    return OMK_OK;
}

int omk_adamw_destroy(omk_adamw *o) {
    if (!o) return OMK_OK;
    {
        OnDevice on(o->l->device);
        if (o->memory) (void)hipFree(o->memory);  // (waits for the device)
        (void)hipGetLastError();
    }
    if (--o->l->children == 0 && o->l->released) delete o->l;
    delete o;
    return OMK_OK;
}

int omk_adamw_create(omk_learner *l, const omk_adamw_desc *desc, omk_adamw **out) try {
    const char *who = "omk_adamw_create";
    if (!l || !desc || !out || (desc->n_tensors > 0 && !desc->h_tensors))
        return learn_fail(OMK_ERR_INVALID, "%s: null argument", who);
    if (desc->n_tensors < 0 || desc->n_tensors > 1 << 24)
        return learn_fail(OMK_ERR_INVALID, "%s: %d tensors", who, desc->n_tensors);
    const int pt = desc->param_type, gt = desc->grad_type, ct = desc->copy_type, st = desc->state_type;
    if (!float_type(pt)) return learn_fail(OMK_ERR_INVALID, "%s: parameters of type %d", who, pt);
    if (!float_type(gt)) return learn_fail(OMK_ERR_INVALID, "%s: gradients of type %d", who, gt);
    if (ct != OMK_NONE && ct != OMK_BF16 && ct != OMK_F16)
        return learn_fail(OMK_ERR_INVALID, "%s: copies of type %d", who, ct);
    if (st != OMK_F32 && st != OMK_F8) return learn_fail(OMK_ERR_INVALID, "%s: states of type %d", who, st);
    if (pt != OMK_F32 && gt != OMK_F32 && gt != pt)
        return learn_fail(OMK_ERR_UNSUPPORTED, "%s: 16-bit parameters with gradients of the other 16-bit type", who);
    if (pt != OMK_F32 && ct != OMK_NONE)
        return learn_fail(OMK_ERR_UNSUPPORTED, "%s: a copy is kept of 32-bit parameters only", who);
    if (!(desc->beta1 >= 0.0 && desc->beta1 < 1.0) || !(desc->beta2 >= 0.0 && desc->beta2 < 1.0) || !(desc->eps >= 0.0) ||
        !((float)desc->eps <= 3e38f) || (desc->eps > 0.0 && desc->eps < 0x1p-126))
        return learn_fail(OMK_ERR_INVALID, "%s: betas %g and %g (0 <= beta < 1), eps %g (0 or at least 2^-126)", who, desc->beta1, desc->beta2,
                          desc->eps);
    std::vector<AdamTensor> tensors((size_t)desc->n_tensors);
    std::vector<int64_t> first_chunk((size_t)desc->n_tensors + 1, 0), elements((size_t)desc->n_tensors);
    int64_t units = 0, n_chunks = 0;
    for (int32_t i = 0; i < desc->n_tensors; i++)
        units += std::max((int64_t)0, std::min(desc->h_tensors[i].n, (int64_t)1 << 40) / kUnit);
    const int32_t chunk_units = units < kManyUnits ? kFewUnits : kChunkUnits;
    units = 0;
    for (int32_t i = 0; i < desc->n_tensors; i++) {
        const omk_adamw_tensor &t = desc->h_tensors[i];
        if (t.n < 0 || t.n > (int64_t)1 << 40) return learn_fail(OMK_ERR_INVALID, "%s: tensor %d of %lld elements", who, i, (long long)t.n);
        if (!std::isfinite(t.lr_scale) || !std::isfinite(t.weight_decay))
            return learn_fail(OMK_ERR_INVALID, "%s: tensor %d: lr_scale %g, weight_decay %g", who, i, t.lr_scale, t.weight_decay);
        if (t.n && (!t.d_param || !t.d_m || !t.d_v || (ct != OMK_NONE && !t.d_copy) ||
                    (st == OMK_F8 && (!t.d_m_scale || !t.d_v_scale))))
            return learn_fail(OMK_ERR_INVALID, "%s: tensor %d: null argument", who, i);
        if (ct == OMK_NONE && t.d_copy)
            return learn_fail(OMK_ERR_INVALID, "%s: tensor %d has a copy, but copies have no type", who, i);
        if (!aligned(t.d_param, width_of(pt)) || !aligned(t.d_copy, 2) || !aligned(t.d_m, width_of(st)) ||
            !aligned(t.d_v, width_of(st)) || (st == OMK_F8 && (!aligned(t.d_m_scale, 4) || !aligned(t.d_v_scale, 4))))
            return learn_fail(OMK_ERR_INVALID, "%s: tensor %d: an address that is no multiple of its type's size", who, i);
        const int64_t own = (t.n + kUnit - 1) / kUnit;
        tensors[i] = AdamTensor{t.n, t.d_param, t.d_copy, t.d_m, t.d_v, t.d_m_scale, t.d_v_scale, units,
                                (float)t.lr_scale, (float)t.weight_decay,
                                aligned(t.d_param, 4 * width_of(pt)) && aligned(t.d_copy, 8) &&
                                    aligned(t.d_m, 4 * width_of(st)) && aligned(t.d_v, 4 * width_of(st))};
        elements[i] = t.n;
        first_chunk[i] = n_chunks;
        units += own;
        n_chunks += (own + chunk_units - 1) / chunk_units;
    }
    first_chunk[(size_t)desc->n_tensors] = n_chunks;
    if (units > UINT32_MAX || n_chunks > INT32_MAX)
        return learn_fail(OMK_ERR_CAPACITY, "%s: over 2^40 elements", who);
    // Every element is stepped once: what is stepped lies at one place each.
    std::vector<std::pair<uintptr_t, uintptr_t>> places;
    places.reserve((size_t)desc->n_tensors * 6);
    for (const AdamTensor &t : tensors) {
        const int64_t n = t.n, scales = (n + kUnit - 1) / kUnit * 4;
        const std::pair<const void *, int64_t> all[] = {{t.param, n * width_of(pt)}, {t.copy, n * 2}, {t.m, n * width_of(st)},
                                                        {t.v, n * width_of(st)}, {t.m_scale, scales}, {t.v_scale, scales}};
        for (int i = 0; i < (st == OMK_F8 ? 6 : 4); i++)
            if (n && all[i].first) places.emplace_back((uintptr_t)all[i].first, (uintptr_t)all[i].first + (uintptr_t)all[i].second);
    }
    std::sort(places.begin(), places.end());
    for (size_t i = 1; i < places.size(); i++)
        if (places[i].first < places[i - 1].second)
            return learn_fail(OMK_ERR_INVALID, "%s: tensors that overlap at %p", who, (const void *)places[i].first);
    std::vector<AdamChunk> chunks((size_t)n_chunks);
    for (int32_t i = 0; i < desc->n_tensors; i++)
        for (int64_t c = first_chunk[i]; c < first_chunk[i + 1]; c++)
            chunks[(size_t)c] = AdamChunk{i, (int32_t)(c - first_chunk[i])};
    omk_adamw *o = new (std::nothrow) omk_adamw();
    if (!o) return learn_fail(OMK_ERR_INVALID, "out of host memory");
    o->l = l;
    l->children++;
    o->n_tensors = desc->n_tensors;
    o->param_type = pt;
    o->grad_type = gt;
    o->copy_type = ct;
    o->state_type = st;
    o->beta1 = desc->beta1;
    o->beta2 = desc->beta2;
    o->eps = desc->eps;
    o->seed = desc->seed;
    o->chunk_units = chunk_units;
    o->first_chunk.swap(first_chunk);
    o->elements.swap(elements);
    OnDevice on(l->device);
    const size_t at_done = 256, at_tensors = at_done + kCountGroups * kCountStep * 4;
    const size_t at_chunks = at_tensors + (tensors.size() * sizeof(AdamTensor) + 255) / 256 * 256;
    hipError_t e = on.status;
    if (e == hipSuccess) e = hipMalloc((void **)&o->memory, at_chunks + chunks.size() * sizeof(AdamChunk) + 16);
    if (e == hipSuccess) {
        o->count = (AdamCount *)o->memory;
        o->done = (uint32_t *)(o->memory + at_done);
        o->tensors = (AdamTensor *)(o->memory + at_tensors);
        o->chunks = (AdamChunk *)(o->memory + at_chunks);
        if (!tensors.empty())
            e = hipMemcpy(o->tensors, tensors.data(), tensors.size() * sizeof(AdamTensor), hipMemcpyHostToDevice);
    }
    if (e == hipSuccess && !chunks.empty())
        e = hipMemcpy(o->chunks, chunks.data(), chunks.size() * sizeof(AdamChunk), hipMemcpyHostToDevice);
    if (e == hipSuccess) e = launch_adamw_set(o->count, o->done, 0, o->beta1, o->beta2, l->stream);
    if (e == hipSuccess) e = hipStreamSynchronize(l->stream);
    if (e != hipSuccess) {
        const int rc = learn_fail(OMK_ERR_HIP, "%s: %s", who, hipGetErrorString(e));
        omk_adamw_destroy(o);
        return rc;
    }
    *out = o;
    return OMK_OK;
} LEARN_NO_THROW

int omk_adamw_step(omk_adamw *o, const void *const *h_grads, double lr, const float *d_lr, const float *d_grad_scale) {
    const char *who = "omk_adamw_step";
    if (o && o->l->released) return learn_fail(OMK_ERR_STATE, "%s: the learner has been destroyed", who);
    if (!o || (o->n_tensors && !h_grads)) return learn_fail(OMK_ERR_INVALID, "%s: null argument", who);
    if (!d_lr && !std::isfinite(lr)) return learn_fail(OMK_ERR_INVALID, "%s: lr %g", who, lr);
    if (!aligned(d_lr, 4) || !aligned(d_grad_scale, 4))
        return learn_fail(OMK_ERR_INVALID, "%s: an address that is no multiple of its type's size", who);
    for (int32_t i = 0; i < o->n_tensors; i++)
        if (!aligned(h_grads[i], width_of(o->grad_type)))
            return learn_fail(OMK_ERR_INVALID, "%s: gradient %d at an address that is no multiple of its type's size", who, i);
    OnDevice on(o->l->device);
    LEARN_TRY(on.status);
    AdamStep s;
    s.tensors = o->tensors;
    s.count = o->count;
    s.done = o->done;
    s.chunk_units = o->chunk_units;
    s.d_lr = d_lr;
    s.d_grad_scale = d_grad_scale;
    s.lr = lr;
    s.beta1 = o->beta1;
    s.beta2 = o->beta2;
    s.eps = (float)o->eps;
    s.seed = o->seed;
    for (int32_t t = 0; t == 0 || t < o->n_tensors; t += kGradsPerLaunch) {
        const int32_t n = std::min(o->n_tensors - t, (int32_t)kGradsPerLaunch);
        AdamGrads g;
        memset(&g, 0, sizeof(g));
        for (int32_t i = 0; i < n; i++) g.g[i] = h_grads[t + i];
        s.first_tensor = t;
        s.chunks = o->chunks + o->first_chunk[t];
        s.n_chunks = o->first_chunk[t + n] - o->first_chunk[t];
        s.last = t + kGradsPerLaunch >= o->n_tensors;
        LEARN_TRY(launch_adamw(o->param_type, o->grad_type, o->copy_type, o->state_type, s, g, o->l->stream));
    }
    return OMK_OK;
}

int omk_adamw_set_steps(omk_adamw *o, int64_t steps) {
    const char *who = "omk_adamw_set_steps";
    if (!o) return learn_fail(OMK_ERR_INVALID, "%s: null argument", who);
    if (o->l->released) return learn_fail(OMK_ERR_STATE, "%s: the learner has been destroyed", who);
    if (steps < 0 || steps > INT32_MAX) return learn_fail(OMK_ERR_INVALID, "%s: %lld steps", who, (long long)steps);
    OnDevice on(o->l->device);
    LEARN_TRY(on.status);
    LEARN_TRY(launch_adamw_set(o->count, o->done, steps, std::pow(o->beta1, (double)steps + 1.0), std::pow(o->beta2, (double)steps + 1.0),
                               o->l->stream));
    return OMK_OK;
}

int omk_adamw_get_steps(omk_adamw *o, int64_t *h_steps) {
    if (!o || !h_steps) return learn_fail(OMK_ERR_INVALID, "omk_adamw_get_steps: null argument");
    if (o->l->released) return learn_fail(OMK_ERR_STATE, "omk_adamw_get_steps: the learner has been destroyed");
    OnDevice on(o->l->device);
    LEARN_TRY(on.status);
    AdamCount c;
    LEARN_TRY(hipMemcpyAsync(&c, o->count, sizeof(c), hipMemcpyDeviceToHost, o->l->stream));
    LEARN_TRY(hipStreamSynchronize(o->l->stream));
    *h_steps = c.steps;
    return OMK_OK;
}

}  // extern "C"
