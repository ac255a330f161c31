"""Products with weights in 8-bit floating point (trc_hip_fp8_*) against 64 bits.

The quantizer is held to every bit: scales are powers of two, so a code is the nearest one to a number that both sides
have exactly.

Products, with u = 2^-24 and S the sum of the terms' magnitudes. In binary16 with sums in 32 bits every product is
exact; a block's 128 are added in 32 bits (an error of 128 u S at most), scaled (2 u), and the blocks and parts added
(a rounding each): (128 + blocks + 16) u S. On the 8-bit instruction eight products are added with at least 12
bits below the largest, so each loses less than 2^-12 of it where it loses any: 7 2^-12 S, and the rest as before.
Each result is rounded once more to its type. What of the terms is taken at all is held to every bit by inputs of
small whole numbers, which all of these add without a rounding."""
import ctypes as C

import numpy as np
import pytest

import fp8_util as F
from conftest import announce
from gpu_util import Dev, Stream, runtime
from traincpp_amd import hip as H
from tuning_util import TYPES, U32, Mat, decode, encode

pytestmark = pytest.mark.gpu

HALF = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 1e-38, "f16": 2.0 ** -25, "bf16": 1e-38}


# ------------------------------------------------------------------ the quantizer

def quantized(x, kind, by_blocks, pad=0, lead=0, extra=0, stream=None):
    """x (raw elements [R, K]) through the device: codes and scale bytes."""
    R, K = x.shape
    kb, rb = -(-K // 128), -(-R // 128) if by_blocks else R
    m = Mat(x, TYPES[kind], pad, lead)
    out = F.Fp8(np.full((R, kb * 128), 0x55, np.uint8), np.full((rb, kb), 0x55, np.uint8), K, extra, lead)
    H.fp8_quantize(m.t, out.t, stream)
    H.sync(stream)
    q, s = out.q.read(), out.s.read()
    out.free()
    m.free()
    return q, s[:, :kb]


def check_quantizer(x, kind, by_blocks=False, **kw):
    q, s = quantized(x, kind, by_blocks, **kw)
    wq, ws = F.quantize(decode(x, kind), by_blocks)
    assert np.array_equal(s, ws), "scales"
    nan = np.isnan(F.VALUES[wq])
    assert np.array_equal(np.isnan(F.VALUES[q]), nan)
    assert np.array_equal(q[~nan], wq[~nan]), "codes"


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("R,K", [(1, 1), (3, 7), (2, 128), (5, 129), (1, 511), (4, 512), (7, 513), (33, 1000), (128, 256),
                                 (129, 385), (300, 2050), (1500, 24600)])
def test_quantizer(hip, kind, R, K):
    announce(f"fp8 quantize {kind} {R}x{K}")
    rng = np.random.default_rng(R * 7 + K)
    x, _ = encode(rng.standard_normal((R, K)) * np.exp(rng.standard_normal((R, 1)) * 2), kind)
    check_quantizer(x, kind)
    if R * K < 1 << 21:
        check_quantizer(x, kind, by_blocks=True)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("by_blocks", [False, True])
def test_quantizer_layouts(hip, kind, by_blocks):
    announce(f"fp8 quantize layouts {kind} {by_blocks}")
    rng = np.random.default_rng(4)
    x, _ = encode(rng.standard_normal((139, 333)), kind)
    for pad, lead, extra in ((1, 1, 0), (3, 5, 1), (8, 3, 2)):
        check_quantizer(x, kind, by_blocks, pad=pad, lead=lead, extra=extra)


@pytest.mark.parametrize("by_blocks", [False, True])
def test_quantizer_rounding(hip, by_blocks):
    """Ties, the scale's borders, blocks of zeros, subnormal and huge values, values that are not finite."""
    announce(f"fp8 quantize rounding {by_blocks}")
    ties = np.concatenate([(F._POSITIVE[1:] + F._POSITIVE[:-1]) / 2, [448.0, 0.0]])
    rows = [np.resize(np.concatenate([ties, -ties]), 256)]
    for top in (448.0, np.nextafter(np.float32(448), np.float32(500)), 449.0, 511.9, 512.0, 1.75, 1.7500001, 2.0 ** -118, 2.0 ** -119,
                2.0 ** -126, 1e-40, 1e-45, 3.4e38, np.finfo(np.float32).max):
        r = np.zeros(256)
        r[3], r[9], r[200] = top, -top / 3, top
        rows.append(r)
    rows.append(np.zeros(256))
    for bad in (np.inf, -np.inf, np.nan):
        r = np.linspace(-2, 2, 256)
        r[5] = bad
        rows.append(r)
    rows.append(np.full(256, np.nan))
    for r in rows:
        x = np.asarray([r] * (130 if by_blocks else 2), np.float32)
        if by_blocks:
            x[1:] *= np.float32(0.5)
        check_quantizer(x, "f32", by_blocks)


# ------------------------------------------------------------------ products

def problem(K, M, N, scales, seed, whole=False, spread=0.3):
    """A weight and activations: codes and scales, as they are held."""
    rng = np.random.default_rng(seed)
    kb, mb = -(-K // 128), -(-M // 128)
    if whole:  # whole numbers from -2 to 2, most of them 0
        draw = lambda r, c: F.encode(rng.choice([0, 0, 0, 1, -1, 2, -2], (r, c)).astype(float))
        w, x = draw(M, K), draw(N, K)
        ws = rng.choice([127, 128, 126], (mb, kb)).astype(np.uint8)
        if scales == "float":
            ws = (2.0 ** (ws.astype(float) - 127) * rng.choice([1, 3], (mb, kb))).astype(np.float32)
        return w, ws, x, rng.choice([127, 128, 126], (N, kb)).astype(np.uint8)
    wv = rng.standard_normal((M, K)) * np.exp(rng.standard_normal((M, 1)) * spread) / np.sqrt(K)
    w, ws = F.quantize(wv, True)
    if scales == "float":
        ws = (2.0 ** (ws.astype(np.float64) - 127) * rng.uniform(0.6, 1.4, ws.shape)).astype(np.float32)
    x, xs = F.quantize(rng.standard_normal((N, K)) * np.exp(rng.standard_normal((1, K)) * spread))
    return w, ws, x, xs


class Product:
    """One product on the device: forward (x is [N, K]) or back (x is dy [N, M])."""

    def __init__(self, w, ws, x, xs, K, M, kind, back=False, extra=0, lead=0, pad=0):
        self.K, self.M, self.N, self.kind, self.back = K, M, x.shape[0], kind, back
        self.w = F.Fp8(w, ws, K, extra, lead)
        self.x = F.Fp8(x, xs, M if back else K, extra, lead)
        dt = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[kind]
        out = np.zeros((self.N, K if back else M), dt)
        self.y = Mat(out, TYPES[kind], pad, lead)

    def run(self, stream=None):
        (H.fp8_mul_mat_back if self.back else H.fp8_mul_mat)(self.w.t, self.x.t, self.y.t, stream)

    def read(self, stream=None):
        H.sync(stream)
        return self.y.read()

    def want(self):
        w = F.values(self.w.codes, self.w.scales, self.K, True)
        x = F.values(self.x.codes, self.x.scales, self.M if self.back else self.K, False)
        b = w if self.back else w.T
        return x @ b, np.abs(x) @ np.abs(b)

    def free(self):
        for b in (self.w, self.x, self.y):
            b.free()


def bound(p, want, mag, fast):
    blocks = -(-(p.M if p.back else p.K) // 128)
    err = (128 + blocks + 16) * U32 * mag
    if fast:
        err += 7 * 2.0 ** -12 * mag
    return err + HALF[p.kind] * (np.abs(want) + err) + TINY[p.kind]


def check(p, fast, got=None):
    if got is None:
        p.run()
        got = p.read()
    want, mag = p.want()
    over = np.abs(decode(got, p.kind) - want) / bound(p, want, mag, fast)
    assert over.max() <= 1, f"{over.max()} of the bound at {np.unravel_index(over.argmax(), over.shape)}"
    return got


def is_fast(p):
    return p.kind != "f32" and (p.back or p.N > H.FP8_MATVEC_MAX_N)


SHAPES = [(1, 1, 1), (128, 16, 1), (127, 17, 3), (300, 5, 16), (513, 130, 17), (640, 33, 33), (1025, 257, 64), (768, 288, 1),
          (128, 128, 65), (129, 64, 66), (1, 200, 100), (700, 300, 129), (2050, 190, 333), (260, 1030, 1100),
          (520, 4100, 4100), (4100, 260, 70)]


@pytest.mark.parametrize("scales", ["pow2", "float"])
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("K,M,N", SHAPES)
@pytest.mark.parametrize("back", [False, True])
def test_whole_numbers(hip, K, M, N, kind, scales, back):
    """Every term is taken once, with its scale: bit for bit."""
    if back:
        K, M = M, K
    announce(f"fp8 whole numbers K={K} M={M} N={N} {kind} {scales} back={back}")
    w, ws, x, xs = problem(K, M, N, scales, K + M + N, whole=True)
    if back:
        _, _, x, xs = problem(M, 1, N, "pow2", K + N, whole=True)
    p = Product(w, ws, x, xs, K, M, kind, back)
    p.run()
    got, want = p.read(), p.want()[0]
    assert np.array_equal(decode(got, kind), encode(want, kind)[1])
    p.free()


@pytest.mark.parametrize("scales", ["pow2", "float"])
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("K,M,N", SHAPES[3:])
@pytest.mark.parametrize("back", [False, True])
def test_products(hip, K, M, N, kind, scales, back):
    if back:
        K, M = M, K
    announce(f"fp8 product K={K} M={M} N={N} {kind} {scales} back={back}")
    w, ws, x, xs = problem(K, M, N, scales, 2 * K + M + N)
    if back:
        x, xs = F.quantize(np.random.default_rng(N).standard_normal((N, M)) * 1e-3)
    p = Product(w, ws, x, xs, K, M, kind, back)
    check(p, is_fast(p))
    p.free()


@pytest.mark.parametrize("scales", ["pow2", "float"])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("K,M,N", [(500, 2000, 600), (300, 4097, 1030), (700, 6000, 400), (130, 4225, 250), (1, 2050, 520)])
@pytest.mark.parametrize("back", [False, True])
def test_numbers_of_tiles(hip, K, M, N, kind, scales, back):
    """From one tile of 64 x 64 a CU to one of 128 x 128, with gaps between rows: whole numbers bit for bit, then others."""
    if back:
        K, M = M, K
    announce(f"fp8 tiles K={K} M={M} N={N} {kind} {scales} back={back}")
    for whole, (extra, lead, pad) in ((True, (0, 0, 0)), (False, (1, 1, 3))):
        w, ws, x, xs = problem(K, M, N, scales, K + 2 * M + N, whole=whole)
        if back:
            _, _, x, xs = problem(M, 1, N, "pow2", K + N, whole=whole)
        p = Product(w, ws, x, xs, K, M, kind, back, extra, lead, pad)
        if whole:
            p.run()
            assert np.array_equal(decode(p.read(), kind), encode(p.want()[0], kind)[1])
        else:
            check(p, is_fast(p))
            p.w.q.read(), p.x.q.read()
        p.free()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("N", [3, 40, 80, 300])
def test_layouts(hip, kind, back, N):
    """Gaps between rows of everything, results on odd addresses; what is around them stays."""
    announce(f"fp8 layouts {kind} back={back} N={N}")
    K, M = 391, 277
    for extra, lead, pad in ((1, 1, 1), (2, 3, 5)):
        w, ws, x, xs = problem(K, M, N, "float", N)
        if back:
            x, xs = F.quantize(np.random.default_rng(N).standard_normal((N, M)))
        p = Product(w, ws, x, xs, K, M, kind, back, extra, lead, pad)
        check(p, is_fast(p))
        p.w.q.read(), p.x.q.read()
        p.free()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("xkind", list(TYPES))
@pytest.mark.parametrize("K,M,N", [(1, 1, 1), (768, 288, 1), (4096, 100, 2), (1000, 77, 4), (1000, 77, 5), (3000, 50, 17), (513, 130, 64),
                                   (24600, 40, 3)])
def test_matvec(hip, kind, xkind, K, M, N):
    """The single-token form: what the quantizer and the product make together, bit for bit."""
    announce(f"fp8 matvec {kind} from {xkind} K={K} M={M} N={N}")
    for scales, pad, lead in (("pow2", 0, 0), ("float", 3, 1)):
        w, ws, _, _ = problem(K, M, 1, scales, K + N)
        rng = np.random.default_rng(K + M)
        raw, v = encode(rng.standard_normal((N, K)) * np.exp(rng.standard_normal((N, 1))), xkind)
        x, xs = F.quantize(v)
        p = Product(w, ws, x, xs, K, M, kind, pad=pad, lead=lead)
        both = check(p, False)
        m = Mat(raw, TYPES[xkind], pad, lead)
        y = Mat(np.zeros_like(both), TYPES[kind], pad, lead)
        H.fp8_matvec(p.w.t, m.t, y.t)
        H.sync()
        assert np.array_equal(y.read(), both)
        for b in (p, m, y):
            b.free()


@pytest.mark.parametrize("K,M,N", [(5000, 100, 1), (14336, 48, 2), (30000, 20, 1), (30000, 33, 2), (4096, 4104, 50), (4096, 4104, 64),
                                   (2048, 14340, 20)])
def test_matvec_of_long_rows_and_large_weights(hip, K, M, N):
    """Several groups of K a wave, activations that do not fit LDS, tiles in parts for few tokens: as above, bit for bit."""
    announce(f"fp8 matvec K={K} M={M} N={N}")
    w, ws, x, xs = problem(K, M, N, "float", K + M + N, whole=True)
    p = Product(w, ws, x, xs, K, M, "f32")
    p.run()
    assert np.array_equal(p.read(), p.want()[0].astype(np.float32))
    rng = np.random.default_rng(N)
    raw = rng.standard_normal((N, K)).astype(np.float32)
    m, y = Mat(raw), Mat(np.zeros((N, M), np.float32))
    H.fp8_quantize(m.t, p.x.t)
    p.run()
    H.fp8_matvec(p.w.t, m.t, y.t)
    H.sync()
    assert np.array_equal(y.read(), p.read())
    for b in (p, m, y):
        b.free()


@pytest.mark.parametrize("K,M,N", [(4096, 14336, 1), (4096, 14336, 2), (4096, 14336, 3), (4100, 14336, 16), (33000, 700, 2), (70000, 64, 64),
                                   (130000, 70, 60)])
def test_matvec_adds_in_the_products_order(hip, K, M, N):
    """Sums that do depend on their order: weights of many rows, and activations that take most of the workspace."""
    announce(f"fp8 order K={K} M={M} N={N}")
    rng = np.random.default_rng(K + M + N)
    kb = -(-K // 128)
    w = rng.integers(0, 127, (M, K), dtype=np.uint8) | rng.integers(0, 2, (M, K), dtype=np.uint8) << 7
    ws = rng.uniform(0.6, 1.4, (-(-M // 128), kb)).astype(np.float32)
    p = Product(w, ws, np.zeros((N, K), np.uint8), np.full((N, kb), 127, np.uint8), K, M, "f32")
    m, y = Mat(rng.standard_normal((N, K)).astype(np.float32)), Mat(np.zeros((N, M), np.float32))
    H.fp8_quantize(m.t, p.x.t)
    p.run()
    H.fp8_matvec(p.w.t, m.t, y.t)
    H.sync()
    assert np.array_equal(y.read(), p.read())
    for b in (p, m, y):
        b.free()


def test_values_that_are_not_finite(hip):
    """A NaN of a token reaches every result of that token and no other; one of the weight every token's result of its row."""
    announce("fp8 not finite")
    for N in (2, 30, 100, 400):
        for kind in TYPES:
            K, M = 300, 290
            w, ws, x, xs = problem(K, M, N, "float", 5)
            x[1, 7] = 127
            w[37, 290] = 255
            p = Product(w, ws, x, xs, K, M, kind)
            p.run()
            got = np.isnan(decode(p.read(), kind))
            want = np.zeros((N, M), bool)
            want[1], want[:, 37] = True, True
            assert np.array_equal(got, want), (N, kind)
            p.free()
            g, gs = F.quantize(np.random.default_rng(3).standard_normal((N, M)))
            w[37, 290] = 0
            g[1, 288] = 127
            w[3, 200] = 127
            p = Product(w, ws, g, gs, K, M, kind, back=True)
            p.run()
            got = np.isnan(decode(p.read(), kind))
            want = np.zeros((N, K), bool)
            want[1], want[:, 200] = True, True
            assert np.array_equal(got, want), (N, kind, "back")
            p.free()


def test_scales_far_apart(hip):
    """Exponents at the ends of what a byte holds: the products stay exact, and overflow only where the result does."""
    announce("fp8 far scales")
    for N in (3, 100):
        for scales in ("pow2", "float"):
            K, M = 256, 130
            w, ws, x, xs = problem(K, M, N, "pow2", 9, whole=True)
            ws[:] = 227
            xs[:] = 27  # 2^100 2^-100
            if scales == "float":
                ws = 2.0 ** (ws.astype(np.float64) - 127)
                ws = ws.astype(np.float32)
            for kind in TYPES:
                p = Product(w, ws, x, xs, K, M, kind)
                p.run()
                assert np.array_equal(decode(p.read(), kind), encode(p.want()[0], kind)[1])
                p.free()


def test_gradient_against_differences(hip):
    """The product is linear in x: a step along a direction of codes changes sum(y g) by the gradient's share of it."""
    announce("fp8 differences")
    K, M, N = 390, 270, 90
    w, ws, x, xs = problem(K, M, N, "float", 21)
    g, gs = F.quantize(np.random.default_rng(22).standard_normal((N, M)))
    step, ss = F.quantize(np.random.default_rng(23).standard_normal((N, K)))
    gv, sv = F.values(g, gs, M, False), F.values(step, ss, K, False)
    y = Product(w, ws, step, ss, K, M, "f32")
    dx = Product(w, ws, g, gs, K, M, "f32", back=True)
    a, b = check(y, False).astype(np.float64), check(dx, False).astype(np.float64)
    wv = np.abs(F.values(w, ws, K, True))
    mag = (np.abs(sv) @ wv.T * np.abs(gv)).sum()
    assert abs((a * gv).sum() - (b * sv).sum()) <= 2 * (128 + 4 + 16) * U32 * mag
    y.free()
    dx.free()


# ------------------------------------------------------------------ streams and graphs

@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("K,M,N,back", [(1000, 300, 40, False), (2000, 300, 100, False), (300, 2000, 100, True),
                                        (500, 700, 700, False)])
def test_same_bits_every_time(hip, kind, K, M, N, back):
    announce(f"fp8 same bits {kind} {K} {M} {N} {back}")
    w, ws, x, xs = problem(K, M, N, "pow2", 31)
    if back:
        x, xs = F.quantize(np.random.default_rng(N).standard_normal((N, M)))
    p = Product(w, ws, x, xs, K, M, kind, back)
    p.run()
    first = p.read()
    s = Stream()
    for stream in (None, s.handle, s.handle):
        p.run(stream)
        assert np.array_equal(p.read(stream), first)
    p.free()
    s.close()


def test_captured_calls_replay(hip):
    """A graph of a token's step (quantized on the way), a prompt's (in two calls) and the way back, replayed over changed
    inputs with eager work in between: each replay as the eager calls."""
    announce("fp8 capture")
    rt = runtime()
    K, M, N = 1500, 500, 90
    w, ws, x, xs = problem(K, M, N, "float", 41)
    rng = np.random.default_rng(42)
    g, gs = F.quantize(rng.standard_normal((N, M)))
    fwd, back = Product(w, ws, x, xs, K, M, "f32"), Product(w, ws, g, gs, K, M, "bf16", back=True)
    few = Mat(rng.standard_normal((9, K)).astype(np.float32))
    many = Mat(rng.standard_normal((N, K)).astype(np.float32))
    y = Mat(np.zeros((9, M), np.float32))

    def step(s):
        H.fp8_matvec(fwd.w.t, few.t, y.t, s)
        H.fp8_quantize(many.t, fwd.x.t, s)
        fwd.run(s)
        back.run(s)

    s = Stream()
    step(s.handle)
    H.sync(s.handle)
    graph, exe = C.c_void_p(), C.c_void_p()
    assert rt.hipStreamBeginCapture(C.c_void_p(s.handle), 0) == 0
    try:
        step(s.handle)
    finally:
        rc = rt.hipStreamEndCapture(C.c_void_p(s.handle), C.byref(graph))
    assert rc == 0
    assert rt.hipGraphInstantiate(C.byref(exe), graph, None, None, 0) == 0
    for _ in range(3):
        for m in (few, many):
            m.dev.buf.upload(rng.standard_normal(m.dev.base.shape).astype(np.float32))
        step(None)
        H.sync()
        want = [y.dev.read(), fwd.y.dev.read(), back.y.dev.read()]
        for o in (y, fwd.y, back.y):
            o.dev.buf.upload(o.dev.base)  # as it began
        assert rt.hipGraphLaunch(exe, C.c_void_p(s.handle)) == 0
        H.sync(s.handle)
        for a, o in zip(want, (y, fwd.y, back.y)):
            assert np.array_equal(a.view(np.uint8), o.dev.read().view(np.uint8))
    rt.hipGraphExecDestroy(exe)
    rt.hipGraphDestroy(graph)
    for b in (fwd, back, few, many, y):
        b.free()
    s.close()
