// The linear operators over bf16 rows.
#include "linear_ops.h"

namespace pygho {
PYGHO_LINEAR_TYPE(bf16)
}  // namespace pygho
