// The linear operators over f32 rows (linear_tile.h).
#include "linear_tile.h"

namespace pygho {
PYGHO_LINEAR_TYPE(float)
}  // namespace pygho
