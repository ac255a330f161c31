// Tiles of 256 rows (fp8_mm.h).
#include "fp8_mm.h"

namespace trc_hip {
F8_INSTANCES(256, 256, 2, 4, 1, 2, true)
}  // namespace trc_hip
