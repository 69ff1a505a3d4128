// The linear operators over bf16 rows (linear_tile.h).
#include "linear_tile.h"

namespace pygho {
PYGHO_LINEAR_TYPE(bf16)
}  // namespace pygho
