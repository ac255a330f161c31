// Tiles of 128 rows (fp8_mm.h).
#include "fp8_mm.h"

namespace trc_hip {
F8_INSTANCES(128, 128, 2, 2, 1, 2)
}  // namespace trc_hip
