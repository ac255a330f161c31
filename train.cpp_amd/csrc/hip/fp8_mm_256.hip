// Tiles of 256 x 256 (fp8_mm.h), 8 waves of 128 rows by 64 tokens.
#include "fp8_mm.h"

namespace trc_hip {
F8_INSTANCES(256, 256, 2, 4, true)
}  // namespace trc_hip
