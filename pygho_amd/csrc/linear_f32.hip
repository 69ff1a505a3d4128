// The linear operators over f32 rows.
#include "linear_ops.h"

namespace pygho {
PYGHO_LINEAR_TYPE(float)
}  // namespace pygho
