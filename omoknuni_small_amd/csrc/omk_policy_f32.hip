// The kernels over rows of logits, for logits of type float.
#include "omk_policy_rows.h"

namespace omk {
OMK_POLICY_TYPE(, float)
}  // namespace omk
