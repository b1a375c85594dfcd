// The kernels over rows of logits, for logits of type f16_t.
#include "omk_policy_rows.h"

namespace omk {
OMK_POLICY_TYPE(, f16_t)
}  // namespace omk
