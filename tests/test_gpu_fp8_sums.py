"""Products with 8-bit weights whose results have 16 bits: sums of 32 bits whatever the number of tokens, and nothing read that
the contract leaves open.

The tolerance is test_gpu_fp8.py's of exact products added in 32 bits, (128 + blocks + 16) 2^-24 of the sum of magnitudes,
and the result's rounding, for every type. Where a few codes are far larger than the rest, products added with 12 bits below the largest
of eight are off by up to 2^-11 of that sum: 50 times and more what is allowed here."""
import numpy as np
import pytest

import fp8_util as F
from conftest import announce
from test_gpu_fp8 import Product, check, problem
from traincpp_amd import hip as H
from tuning_util import decode, encode

pytestmark = pytest.mark.gpu

# tiles of 64 x 64, the same in parts, of 128 x 64 and 128 x 128; rows and tokens that fill none; K, M, N
SHAPES = [(32, 70, 65), (128, 200, 100), (2050, 199, 333), (4096, 130, 65), (640, 4096, 512), (300, 4300, 600), (640, 4096, 1100)]


def spiky(rng, rows, cols):
    """Codes of which one in 16 is +-448 and the others lie around 1/4: sums whose largest terms nearly cancel."""
    v = np.where(rng.random((rows, cols)) < 1 / 16, rng.choice([-448.0, 448.0], (rows, cols)), rng.standard_normal((rows, cols)) / 4)
    return F.encode(v)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("K,M,N", SHAPES)
@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("scales", ["pow2", "float"])
def test_sums_are_of_32_bits(hip, K, M, N, kind, back, scales):
    if back:
        K, M = M, K
    announce(f"fp8 sums K={K} M={M} N={N} {kind} {scales} back={back}")
    rng = np.random.default_rng(K + M + N)
    summed = M if back else K
    kb, mb = -(-K // 128), -(-M // 128)
    w, x = spiky(rng, M, K), spiky(rng, N, summed)
    # (scales that keep results within F16's range)
    ws = np.full((mb, kb), 118, np.uint8) if scales == "pow2" else rng.uniform(0.6, 1.4, (mb, kb)).astype(np.float32) * np.float32(2.0 ** -9)
    xs = rng.choice([117, 118], (N, -(-summed // 128))).astype(np.uint8)
    p = Product(w, ws, x, xs, K, M, kind, back)
    check(p, False)
    p.free()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("K,M,N,back", [(2050, 190, 333, False), (4096, 300, 1100, False), (300, 4096, 600, True), (700, 2050, 40, True)])
def test_sums_of_normal_data(hip, K, M, N, back, kind):
    announce(f"fp8 normal K={K} M={M} N={N} {kind} back={back}")
    w, ws, x, xs = problem(K, M, N, "float", K + M)
    if back:
        x, xs = F.quantize(np.random.default_rng(N).standard_normal((N, M)))
    p = Product(w, ws, x, xs, K, M, kind, back)
    check(p, False)
    p.free()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("N", [3, 100, 1100])
@pytest.mark.parametrize("scales", ["pow2", "float"])
def test_scales_are_multiplied_first(hip, N, kind, scales):
    """Tokens near 2^127 under a weight near 2^-126, and the other way round: whole numbers bit for bit, forward and back."""
    announce(f"fp8 scales multiplied N={N} {kind} {scales}")
    for wb, xb in ((1, 254), (254, 1)):
        for back in (False, True):
            K, M = 300, 260
            w, ws, x, xs = problem(K, M, N, "pow2", 9, whole=True)
            if back:
                _, _, x, xs = problem(M, 1, N, "pow2", 10, whole=True)
            ws[:], xs[:] = wb, xb
            if scales == "float":
                ws = np.ldexp(np.float32(1), ws.astype(int) - 127).astype(np.float32)
            p = Product(w, ws, x, xs, K, M, kind, back)
            p.run()
            assert np.array_equal(decode(p.read(), kind), encode(p.want()[0], kind)[1]), (wb, back)
            p.free()
