// What the translation units behind include/omk_learn.h share: arguments of the kernels, and their launchers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/omk_learn.h"

namespace omk {

// Sets the message of omk_last_error (omk_api.hip) and returns the code.
int learn_fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));

struct Rows {
    const void *x;
    int64_t stride;
    int64_t rows;
    int32_t actions;
    int64_t first;  // row of a launch's first block
    const uint32_t *legal;
    int64_t legal_stride;
    int32_t words;  // of a row's mask
    int64_t span;   // elements from the first to behind the last
    bool aligned;   // the first lies at a multiple of 16 bytes
};

// Rows of up to this many actions are held in registers, whatever their type and alignment (65536 and up to 7 elements
// before the row, in the widest team); wider ones need work space.
constexpr int32_t kMostInRegisters = 65536 - 8;
int64_t wide_work(int64_t rows, int32_t actions);  // bytes

struct PolicyLoss {
    const int32_t *moves;
    const float *old_logprob, *advantage, *ref_logprob, *weight;
    double log_low, log_high;  // borders of the ratio's logarithm
    double low, high;          // borders of the ratio
    double kl_weight, scale;
    void *grad;
    int64_t grad_stride;
    float *logprob, *kl;
    double *shares;  // work space: the blocks' shares of the loss (at most one a row), and what wide rows need
    float *loss;
};

struct PreferenceLoss {
    const int32_t *moves, *line_begin;
    int64_t pairs;
    const float *ref_logprob;
    double beta, smoothing, scale;
    void *grad;
    int64_t grad_stride;
    int32_t zero_rest;
    float *margin, *line_logprob, *loss;
    // work space, per row: log-probability of the move (0: left out), largest logit, one over the sum of exponentials,
    // derivative of the loss by the log-probability; per pair: its share of the loss; and what wide rows need
    void *work;
    double *logprob;
    float *top, *inverse, *slope, *pair_loss;
};

hipError_t launch_priors(int type, const Rows &r, float *priors, int64_t prior_stride, void *work, hipStream_t stream);
hipError_t launch_logprobs(int type, const Rows &r, const int32_t *moves, float *logprob, float *entropy, void *work,
                           hipStream_t stream);
hipError_t launch_policy_loss(int type, const Rows &r, const PolicyLoss &p, hipStream_t stream);
// before: bytes of its work space that come before what wide rows need
hipError_t launch_preference_loss(int type, const Rows &r, const PreferenceLoss &p, int64_t before, hipStream_t stream);
hipError_t launch_set_float(float *to, float value, hipStream_t stream);

constexpr int kUnit = 256;      // elements that share a scale, and that a wavefront steps at a time
// Units of a chunk: what a block takes at a time, all of one tensor.  kChunkUnits where there are enough of them to
// fill the card with blocks, kFewUnits (a unit a wavefront) in smaller networks.  With 8-bit moments 1 M weights take
// 13.6 us in chunks of 4 units and 17.1 us in chunks of 32, 4 M weights 31.8 and 28.3 us, 7 M weights 52 and 36 us.
constexpr int kChunkUnits = 32, kFewUnits = 4;
constexpr int64_t kManyUnits = 8192;
constexpr int kGradsPerLaunch = 256;  // gradient pointers that travel as kernel arguments

struct AdamTensor {
    int64_t n;
    void *param, *copy, *m, *v;
    float *m_scale, *v_scale;
    int64_t first_unit;  // units of the tensors before it
    float lr_scale, weight_decay;
    bool vectors;  // all addresses (but the gradient's) are multiples of four elements
};

struct AdamChunk {
    int32_t tensor;
    int32_t chunk;  // of the tensor's
};

// Lives on the device: steps done, and what the next step, t, is made with: beta1^t, beta2^t, 1 / (1 - beta1^t) and
// 1 / sqrt(1 - beta2^t), which every block would have to work out; and the groups of blocks that are done with that step.
struct AdamCount {
    double power1, power2, unbias;
    float root;
    uint32_t done;
    int64_t steps;
};

constexpr int kCountGroups = 64, kCountStep = 32;  // counters of blocks that are done, 128 bytes apart

struct AdamGrads {
    const void *g[kGradsPerLaunch];
};

struct AdamStep {
    const AdamTensor *tensors;
    const AdamChunk *chunks;
    int64_t n_chunks;
    int32_t chunk_units;
    int32_t first_tensor;
    AdamCount *count;
    uint32_t *done;  // the groups' counters, 0 between steps
    const float *d_lr, *d_grad_scale;
    double lr;
    double beta1, beta2;
    float eps;
    uint32_t seed;
    int32_t last;  // this launch ends the step
};

hipError_t launch_adamw(int param, int grad, int copy, int state, const AdamStep &s, const AdamGrads &g,
                        hipStream_t stream);
hipError_t launch_adamw_set(AdamCount *count, uint32_t *done, int64_t steps, double power1, double power2, hipStream_t stream);

}  // namespace omk
