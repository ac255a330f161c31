"""Adapters (trc_hip_lora, trc_hip_lora_back) where every bit of the result is known: values that are not
finite, in each type's own way through the kernels."""
import numpy as np
import pytest

from conftest import announce
from test_gpu_lora import Problem, near, run_forward
from tuning_util import TYPES

pytestmark = pytest.mark.gpu

# quiet and signalling, either sign, with payloads in the upper bits, in the lower 16 alone and everywhere
NANS = [0x7FC00000, 0xFFC00000, 0x7F800001, 0xFF800001, 0x7F80FFFF, 0xFF808000, 0x7F810000, 0x7FFFFFFF]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("K,M,R,lens", [
    (96, 70, 8, [3, 17, 1]),        # K in whole chunks of 32
    (90, 70, 10, [3, 17, 1]),       # and with a rest, a rank that is no whole four
    (4160, 300, 40, [3, 17, 1]),    # h in parts, in a launch of its own
])
def test_every_nan_stays_one(hip, kind, K, M, R, lens):
    """... in h and y of its token, wherever along x it stands, and in no other token's."""
    announce(f"lora NaNs {kind} K={K} R={R}")
    p = Problem(kind, K, M, R, lens, [0, 2, 1])
    good = p.x.copy()
    wh, hm, wy, ym = p.forward(p.base)
    tokens = [1, 5, 19, 20]
    rest = np.setdiff1d(np.arange(p.T), tokens)
    for i, bits in enumerate(NANS):
        p.x = good.copy()
        for j, t in enumerate(tokens):
            p.x.view(np.uint32)[t, (13 * i + 29 * j) % K] = bits
        h, y = run_forward(p)
        assert np.isnan(h[tokens]).all(), f"{bits:#x}: h {h[tokens][~np.isnan(h[tokens])][:4]}"
        assert np.isnan(y[tokens]).all(), f"{bits:#x}: y {y[tokens][~np.isnan(y[tokens])][:4]}"
        near(h[rest], wh[rest], hm[rest], p.K + 2, "h")
        near(y[rest], wy[rest], ym[rest], p.K + p.R + 4, "y")
    p.free()
