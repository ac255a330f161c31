// Tiles of 64 rows (fp8_mm.h).
#include "fp8_mm.h"

namespace trc_hip {
F8_INSTANCES(64, 64, 2, 2, 2, 2)
F8_INSTANCES(64, 64, 2, 2, 2, 3)
}  // namespace trc_hip
