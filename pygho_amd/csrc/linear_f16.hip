// The linear operators over f16 rows (linear_tile.h).
#include "linear_tile.h"

namespace pygho {
PYGHO_LINEAR_TYPE(f16)
}  // namespace pygho
