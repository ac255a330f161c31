"""Adapters (trc_hip_lora, trc_hip_lora_back) where every bit of the result is known: sums of one
product each, and values that are not finite, in each type's own way through the kernels."""
import numpy as np
import pytest

from conftest import announce
from test_gpu_lora import Problem, near, run_backward, run_forward
from traincpp_amd import hip as H
from tuning_util import TYPES, encode

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


def one_term_sums(kind, K, M, R, lens, ids, seed=11, pad=0):
    """A problem whose sums each have one product that is not 0, by a power of two: h, y, g and dx are known to the
    last bit, from factors of 24 bits."""
    p = Problem(kind, K, M, R, lens, ids, seed=seed, pad=pad)
    rng = np.random.default_rng(seed)
    power = lambda: rng.choice([-1.0, 1.0], R) * 2.0 ** rng.integers(-6, 7, R)
    p.a64, p.b64 = np.zeros_like(p.a64), np.zeros_like(p.b64)
    for i in range(p.n):
        p.a64[i, np.arange(R), rng.permutation(K)[:R]] = power()
        p.b64[i, rng.permutation(M)[:R], np.arange(R)] = power()
    t = TYPES[kind]
    for name, w in (("a", p.a64), ("b", p.b64)):
        setattr(p.set, name, p.adapters(np.ascontiguousarray(encode(w, kind)[0]), t, 0))
    p.scale = (2.0 ** rng.integers(-3, 4, p.n)).astype(np.float32)
    p.set.scale = p.vector(p.scale, H.TYPE_F32)
    for x in (p.x, p.dy):  # all 24 bits of a float, of many sizes
        bits = rng.integers(1 << 23, 1 << 24, x.shape) | 1
        x[...] = bits * rng.choice([-1.0, 1.0], x.shape) * 2.0 ** rng.integers(-44, -3, x.shape)
    return p


EXACT = [  # K, M, R, lens, ids
    (32, 64, 4, [16, 1], [0, 1]),
    (64, 70, 8, [3, 1, 30], [0, 2, 1]),
    (256, 192, 16, [20, 1], [1, 0]),
    (96, 160, 24, [40, 5], [2, 0]),            # two tiles of the rank, 16 bytes of a row of B at a time
    (100, 130, 20, [33, 1], [1, 2]),           # eight bytes, a rest of K and of M
    (512, 320, 64, [50, 2, 1], [0, 1, 2]),
    (4096, 640, 32, [70, 3], [2, 0]),          # h in parts, two launches
    (2048, 512, 128, [19, 1, 2], [1, 0, 2]),
    (300, 290, 250, [18, 4], [0, 1]),          # a rank that is no whole four
]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape", EXACT, ids=str)
def test_one_term_sums_are_exact(hip, kind, shape):
    """Nothing of a float factor is left out, whatever instructions a type's products are made on."""
    announce(f"lora exact {kind} {shape}")
    p = one_term_sums(kind, *shape)
    h, y = run_forward(p, use_base=False)
    wh, _, wy, _ = p.forward(np.zeros_like(p.base))
    assert np.array_equal(wh, wh.astype(np.float32)) and np.array_equal(wy, wy.astype(np.float32))
    assert np.array_equal(h, wh), f"h: {np.argwhere(h != wh)[:4].tolist()}"
    assert np.array_equal(y, wy), f"y: {np.argwhere(y != wy)[:4].tolist()}"
    g, dx, da, db = run_backward(p, h, use_base=False, da0=np.zeros(p.a.shape, np.float32), db0=np.zeros(p.b.shape, np.float32))
    (wg, _), (wdx, _), _, _ = p.backward(np.zeros_like(p.dxb), h)
    assert np.array_equal(g, wg), f"g: {np.argwhere(g != wg)[:4].tolist()}"
    assert np.array_equal(dx, wdx), f"dx: {np.argwhere(dx != wdx)[:4].tolist()}"
    # with a base: one more rounding, of the sum
    h, y = run_forward(p)
    assert np.array_equal(y, wy.astype(np.float32) + p.base)
    p.free()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("K,M,R,lens", [(96, 70, 8, [3, 17, 2]), (4160, 300, 40, [3, 17, 2])])
def test_values_that_are_not_finite_in_16_bits(hip, kind, bad, K, M, R, lens):
    """... stay with their token, and those of an adapter with the tokens that use it."""
    announce(f"lora not finite {kind} {bad} K={K}")
    p = Problem(kind, K, M, R, lens, [0, 2, 1])
    wh, hm, wy, ym = p.forward(p.base)
    good = p.x[[1, 6]].copy()
    p.x[1, 7], p.x[6, K - 1] = bad, bad
    h, y = run_forward(p)
    rest = np.setdiff1d(np.arange(p.T), [1, 6])
    assert not np.isfinite(h[[1, 6]]).any() and not np.isfinite(y[[1, 6]]).any()
    near(h[rest], wh[rest], hm[rest], p.K + 2, "h")
    near(y[rest], wy[rest], ym[rest], p.K + p.R + 4, "y")

    p.x[[1, 6]] = good
    a, b = p.a.copy(), p.b.copy()
    value = encode(np.array([bad], np.float32), kind)[0][0] if not np.isnan(bad) else {"f16": np.float16(np.nan), "bf16": np.uint16(0x7FC0)}[kind]
    a[2, 3, 40], b[1, 9, 5] = value, value
    p.set.a, p.set.b = p.adapters(a, TYPES[kind], 0), p.adapters(b, TYPES[kind], 0)
    h, y = run_forward(p)
    first, second, third = slice(0, 3), slice(3, 20), slice(20, 22)
    assert not np.isfinite(h[second, 3]).any() and not np.isfinite(y[second]).any()
    keep = np.arange(R) != 3
    near(h[second][:, keep], wh[second][:, keep], hm[second][:, keep], p.K + 2, "h")
    assert not np.isfinite(y[third, 9]).any()
    keep = np.arange(M) != 9
    near(y[third][:, keep], wy[third][:, keep], ym[third][:, keep], p.K + p.R + 4, "y")
    near(h[third], wh[third], hm[third], p.K + 2, "h")
    near(h[first], wh[first], hm[first], p.K + 2, "h")
    near(y[first], wy[first], ym[first], p.K + p.R + 4, "y")
    p.free()
