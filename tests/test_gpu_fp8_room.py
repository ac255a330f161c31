"""Products with 8-bit weights whose rows of scales have more room than scales: the contract leaves open what those
bytes hold, so no result may depend on them."""
import numpy as np
import pytest

import fp8_util as F
from conftest import announce
from test_gpu_fp8 import Product, problem

pytestmark = pytest.mark.gpu


def fill_room(b, used, value):
    """Bytes `used` to `room` of every row, and what lies between rows."""
    raw = b.dev.read()
    body = raw[b.lead:b.lead + b.x.shape[0] * b.pitch].reshape(-1, b.pitch)
    body[:, used:] = value
    b.dev.buf.upload(raw)


# Numbers of blocks summed over that two groups of waves share unevenly (1, 3, 5, 17) and evenly (4, 32); a few tokens, tiles of
# 64 x 64 in parts, one a CU and more of them, and of 128 x 64.
CASES = [(rows, N, summed, kind) for rows, N in ((190, 3), (190, 70), (300, 333)) for summed in (100, 300, 512, 2050)
         for kind in ("f32", "f16")]
CASES += [(190, 70, 640, "bf16"), (190, 70, 4096, "f32"), (4300, 600, 300, "bf16"), (4300, 600, 2050, "f32"), (900, 1000, 640, "f32"),
          (700, 2600, 300, "f32")]


@pytest.mark.parametrize("scales", ["pow2", "float"])
@pytest.mark.parametrize("rows,N,summed,kind", CASES)
@pytest.mark.parametrize("back", [False, True])
def test_bytes_behind_the_scales(hip, rows, N, summed, scales, kind, back):
    announce(f"fp8 room rows={rows} N={N} summed={summed} {scales} {kind} back={back}")
    K, M = (rows, summed) if back else (summed, rows)
    w, ws, x, xs = problem(K, M, N, scales, summed + rows)
    if back:
        x, xs = F.quantize(np.random.default_rng(N).standard_normal((N, M)))
    ws = np.minimum(ws + 2, 254).astype(np.uint8) if ws.dtype == np.uint8 else ws * 4  # (scales of 2 and more among them)
    p = Product(w, ws, x, xs, K, M, kind, back, extra=1)
    p.run()
    want = p.read()
    for value in (0xFF, 254, 1):
        fill_room(p.x.s, xs.shape[1], value)
        if ws.dtype == np.uint8:
            fill_room(p.w.s, ws.shape[1], value)
        p.run()
        assert np.array_equal(p.read(), want), value
    p.free()
