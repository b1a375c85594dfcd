// The kernels over rows of logits, for logits of type bf16_t.
#include "omk_policy_rows.h"

namespace omk {
OMK_POLICY_TYPE(, bf16_t)
}  // namespace omk
