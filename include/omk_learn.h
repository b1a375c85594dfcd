/*
 * omk_learn.h -- C ABI of what lies between a search and the network that it asks (MI355X / gfx950).
 *
 * A search takes a network's answer (one row of logits over the action space per position) and gives what the
 * network is trained on.  This header is the way from the logits to the priors of omk_expand_batch*
 * (MCTSNode::setPriorProbabilities, src/mcts/mcts_node.cpp:512-593), and from the moves that a search played
 * (omk_forest_action_probabilities) to the gradient by the logits and the step of the weights.
 *
 * Conventions are those of omk_forest.h: omk_status, omk_last_error(), opaque handles, d_* for device pointers,
 * h_* for host pointers, and
 *   - every call is enqueued on the learner's stream (omk_learner_set_stream) and returns; nothing is waited for unless
 *     it says so.  A call allocates nothing but in omk_*_create, keeps nothing of its arguments, and holds no work
 *     space of its own: what it needs the caller passes (d_work).  So calls may be captured into graphs, and
 *     graphs replayed side by side, as long as their buffers differ;
 *   - results and work space lie apart from each other and from all that a call reads; only a gradient by the logits may take
 *     the logits' place.  Calls whose arguments do not are refused;
 *   - a learner's device need not be the calling thread's: calls put the thread's device back;
 *   - one host thread drives a learner (and its optimizers) at a time.
 *
 * Rows.  A row is a position (or a token); its columns are the actions.  A row's legal actions are the set bits of
 * its words in d_legal (bit i of word i/32, as in omk_soa_view.legal), or all of them.  What stands in the columns
 * of illegal actions is never looked at, infinities and NaN included; their probability and gradient are 0.
 * With m = max over the legal x, S = sum exp(x - m):   log p(a) = x_a - m - log S.
 * A row without a legal action, or with -inf in all of them, has no policy: probabilities and entropy are 0.  A row
 * that has no policy, or whose move lies outside [0, actions) (a padded position: -1) or is not legal (or has the
 * logit -inf), is LEFT OUT of a loss: its loss, log-probability and gradient are 0.  A NaN or +inf among the legal
 * logits makes its row's results NaN, in the columns of illegal actions too.
 */
#ifndef OMK_LEARN_H
#define OMK_LEARN_H

#include "omk_forest.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef enum omk_type {
    OMK_F32 = 0,
    OMK_BF16 = 1,
    OMK_F16 = 2,
    OMK_F8 = 3,   /* e4m3 with a scale for each block of 256 (optimizer states only) */
    OMK_NONE = -1 /* where a type is optional */
} omk_type;

#define OMK_MAX_ACTIONS (1 << 24)
#define OMK_MAX_PAIRS (1 << 23)

typedef struct omk_learner omk_learner;
typedef struct omk_adamw omk_adamw;

/* A device and a stream.  A learner starts on its device's default stream. */
int omk_learner_create(int32_t device, omk_learner **out);
int omk_learner_destroy(omk_learner *l);
/* The hipStream_t that the calls from here on are enqueued on (NULL: the device's default stream). */
int omk_learner_set_stream(omk_learner *l, void *hip_stream);
int omk_learner_get_stream(omk_learner *l, void **hip_stream_out);
/* Waits for the learner's stream. */
int omk_learner_sync(omk_learner *l);

typedef struct omk_policy_rows {
    const void *d_logits;    /* row r, action j at element r * row_stride + j */
    int64_t row_stride;      /* elements; at least `actions` when there is more than one row.  What lies between
                                two rows may be read, and is not looked at */
    int64_t rows;            /* 0 .. 2^31 - 1; with 0 every call returns OMK_OK (a loss is then set to 0) */
    int32_t actions;         /* 1 .. OMK_MAX_ACTIONS */
    int32_t type;            /* OMK_F32, OMK_BF16, OMK_F16 */
    const uint32_t *d_legal; /* NULL: every action is legal */
    int64_t legal_stride;    /* words between two rows' masks; 0: one mask for all rows */
} omk_policy_rows;

/* Bytes of d_work that the two calls below need: 0 (and d_work may be NULL) for rows of up to 65528 actions.  Work
 * space lies at a multiple of 16 bytes; the same memory may serve calls one after another on a stream. */
int64_t omk_policy_work(int64_t rows, int32_t actions);

/* Probabilities of the actions, in 32 bits: d_priors[r * prior_stride + j].  What omk_expand_batch takes as
 * h_policy. */
int omk_policy_priors(omk_learner *l, const omk_policy_rows *rows, float *d_priors, int64_t prior_stride, void *d_work,
                      int64_t work_bytes);

/* d_logprob[r] = log-probability of the move d_moves[r]: 0 where the move lies outside [0, actions), -inf where it
 * is not legal or the row has no policy.  d_entropy[r] = -sum p log p.  Either output may be NULL (d_moves too, then,
 * when d_logprob is). */
int omk_policy_logprobs(omk_learner *l, const omk_policy_rows *rows, const int32_t *d_moves, float *d_logprob,
                        float *d_entropy, void *d_work, int64_t work_bytes);

/* Clipped policy loss with a KL term.  Row by row, with lp = log p(move):
 *   ratio = exp(lp - old_logprob)
 *   l     = -min(ratio * advantage, clamp(ratio, 1 - clip_low, 1 + clip_high) * advantage)
 *           + kl_weight * kl,   kl = exp(ref_logprob - lp) - (ref_logprob - lp) - 1
 *   loss  = scale * sum over rows of weight * l
 * and the gradient of the loss by every logit.  (A derivative by lp that passes the 32-bit range is held at its end, so that an
 * illegal action's gradient is 0 beside it too; the loss is infinite there.)  An advantage of 0 gives no loss at whatever ratio, and a row of weight 0
 * adds nothing to loss and gradient, whatever its other columns hold. */
typedef struct omk_policy_samples {
    const int32_t *d_moves;
    const float *d_old_logprob;
    const float *d_advantage;
    const float *d_ref_logprob; /* NULL: no KL term (kl_weight must be 0) */
    const float *d_weight;      /* NULL: 1 */
} omk_policy_samples;
typedef struct omk_policy_loss_params {
    double clip_low;  /* >= 0 */
    double clip_high; /* >= 0 */
    double kl_weight; /* >= 0 */
    double scale;     /* finite; 1 / rows for a mean */
} omk_policy_loss_params;
typedef struct omk_policy_loss_out {
    float *d_loss;       /* one value */
    void *d_grad;        /* as the logits' type; the logits themselves are allowed (same stride); NULL: no gradient */
    int64_t grad_stride; /* elements */
    float *d_logprob;    /* [rows]; 0 in rows left out */
    float *d_kl;         /* [rows]; 0 in rows left out; NULL allowed */
} omk_policy_loss_out;
/* Bytes of d_work for this many rows. */
int64_t omk_policy_loss_work(int64_t rows, int32_t actions);
int omk_policy_loss(omk_learner *l, const omk_policy_rows *rows, const omk_policy_samples *samples,
                    const omk_policy_loss_params *params, const omk_policy_loss_out *out, void *d_work,
                    int64_t work_bytes);

/* Preference loss over pairs of lines of play.  Line s is the rows d_line_begin[s] .. d_line_begin[s+1] - 1; of
 * the lines 2k and 2k + 1 the first is preferred.  With S_s the sum of a line's log-probabilities (rows left out
 * count nothing) and u_k = beta * ((S_2k - ref_2k) - (S_2k+1 - ref_2k+1)):
 *   loss = scale * sum over pairs of -(1 - label_smoothing) log sigmoid(u) - label_smoothing log sigmoid(-u)
 * d_ref_logprob[s] = the line's sum under the reference policy (NULL: 0); a call without d_grad on the reference's logits
 * gives it as d_line_logprob.  d_line_begin must not decrease.  (Bounds that do not fit
 * are taken as the nearest that do: the first and the last inside [0, rows], the others between these two; a line that would end before it begins is
 * empty; which line's gradient a row of two lines gets is open.)  Rows before the first line and behind the last are not
 * read.  0 .. OMK_MAX_PAIRS pairs; with 0 the loss is 0, and every row is a row of no line (zero_rest). */
typedef struct omk_preference_params {
    double beta;
    double label_smoothing; /* 0 .. 0.5 */
    double scale;           /* finite; 1 / pairs for a mean */
} omk_preference_params;
typedef struct omk_preference_out {
    float *d_loss;         /* one value */
    void *d_grad;          /* as in omk_policy_loss_out */
    int64_t grad_stride;
    float *d_margin;       /* [pairs] u; NULL allowed */
    float *d_line_logprob; /* [2 * pairs] S; NULL allowed */
    int32_t zero_rest;     /* gradients of rows of no line: 0 = left as they are, 1 = set to 0 */
} omk_preference_out;
int64_t omk_preference_loss_work(int64_t rows, int32_t actions, int64_t pairs);
int omk_preference_loss(omk_learner *l, const omk_policy_rows *rows, const int32_t *d_moves,
                        const int32_t *d_line_begin, int64_t pairs, const float *d_ref_logprob,
                        const omk_preference_params *params, const omk_preference_out *out, void *d_work,
                        int64_t work_bytes);

/* AdamW over many tensors at once.  Step t (the optimizer counts), element by element, in 32 bits:
 *   g = grad * grad_scale;  m = beta1 m + (1 - beta1) g;  v = beta2 v + (1 - beta2) g g
 *   p = p - lr lr_scale weight_decay p - lr lr_scale / (1 - beta1^t) * m / (sqrt(v / (1 - beta2^t)) + eps)
 * With states in 8 bits d_m and d_v hold e4m3 codes of m and of sqrt(v), with a 32-bit scale for each 256 elements
 * of the tensor (its last block may be shorter); the largest magnitude of a block becomes 448, and the others are
 * rounded up or down at random with the probability of their place between two codes (random numbers from seed, t and
 * the element's place, so a run repeats): to the nearest, a second moment that changes by a thousandth a step would
 * never leave its code.  A sqrt(v) that is not 0 keeps the smallest code at least.
 * An infinite gradient or a NaN stays in the moments, as in the formula, and with states in 8 bits in those of all 256 elements
 * that share its scale: look at gradients before the step (a step is not left out on the device). */
typedef struct omk_adamw_tensor {
    int64_t n;
    void *d_param;
    void *d_copy; /* the parameter in copy_type, written with every step; NULL where copy_type is OMK_NONE */
    void *d_m, *d_v;
    float *d_m_scale, *d_v_scale; /* OMK_F8: ceil(n / 256) each */
    double lr_scale, weight_decay;
} omk_adamw_tensor;
typedef struct omk_adamw_desc {
    int32_t n_tensors;
    const omk_adamw_tensor *h_tensors;
    int32_t param_type; /* OMK_F32, OMK_BF16, OMK_F16 */
    int32_t grad_type;  /* OMK_F32, or param_type, or with 32-bit parameters either 16-bit type */
    int32_t copy_type;  /* OMK_NONE, or with 32-bit parameters OMK_BF16 or OMK_F16 */
    int32_t state_type; /* OMK_F32, OMK_F8 */
    double beta1, beta2;
    double eps; /* 0, or 2^-126 and more */
    uint32_t seed;
} omk_adamw_desc;
/* Copies the description to the device; the tensors stay the caller's, and where they are.  Pointers need the alignment of
 * their type only; two that overlap are refused, a tensor that is there twice among them.  Waits for the copy. */
int omk_adamw_create(omk_learner *l, const omk_adamw_desc *desc, omk_adamw **out);
/* Waits for the device.  (An optimizer whose learner has been destroyed only waits to be destroyed itself.) */
int omk_adamw_destroy(omk_adamw *o);
/* One step.  h_grads[i]: tensor i's gradient in device memory, or NULL: that tensor is left as it is.
 * d_grad_scale: NULL, or a 32-bit value in device memory that gradients are multiplied by (a clipping factor, one over a loss
 * scale).  d_lr: NULL, or the learning rate in device memory, taken in the place of `lr` (for replayed graphs).
 * The count t lives on the device, and a replayed step counts too. */
int omk_adamw_step(omk_adamw *o, const void *const *h_grads, double lr, const float *d_lr, const float *d_grad_scale);
/* Steps done.  set: in stream order (0 .. 2^31 - 1).  get: waits for the stream. */
int omk_adamw_set_steps(omk_adamw *o, int64_t steps);
int omk_adamw_get_steps(omk_adamw *o, int64_t *h_steps);

#ifdef __cplusplus
}
#endif
#endif
