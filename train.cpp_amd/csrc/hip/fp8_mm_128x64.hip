// Tiles of 128 rows by 64 tokens (fp8_mm.h).
#include "fp8_mm.h"

namespace trc_hip {
F8_INSTANCES(128, 64, 2, 2, 2, 3)
}  // namespace trc_hip
