// Tiles of 64 x 64 (fp8_mm.h), 4 waves of 32 rows by 32 tokens.
#include "fp8_mm.h"

namespace trc_hip {
F8_INSTANCES(64, 64, 2, 2, true)
F8_INSTANCES(64, 64, 2, 2, false)
}  // namespace trc_hip
