// The linear operators over f16 rows.
#include "linear_ops.h"

namespace pygho {
PYGHO_LINEAR_TYPE(f16)
}  // namespace pygho
