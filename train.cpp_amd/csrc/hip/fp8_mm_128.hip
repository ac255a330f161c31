// Tiles of 128 x 128 (fp8_mm.h), 4 waves of 64 rows by 64 tokens.
#include "fp8_mm.h"

namespace trc_hip {
F8_INSTANCES(128, 128, 2, 2, true)
F8_INSTANCES(128, 128, 2, 2, false)
}  // namespace trc_hip
