"""Adapters of many requests (trc_hip_lora) and their gradients (trc_hip_lora_back)
against plain sums in 64 bits.

Tolerance: a sum of n products in 32 bits is rounded n times, each time by at most 2^-24
of a partial sum, which no partial sum of the products' magnitudes is below. Taken as
independent, the roundings of n terms add up to more than 8 sqrt(n) times that with a probability
under 2e-13 (Hoeffding), so 8 sqrt(n) 2^-24 times the sum of magnitudes bounds each element; two sums
in a row have n of both."""
import ctypes as C

import numpy as np
import pytest

from conftest import announce
from gpu_util import Dev, Stream, runtime
from traincpp_amd import hip as H
from tuning_util import TYPES, U32, Mat, encode, starts, vec

pytestmark = pytest.mark.gpu


class Problem:
    def __init__(self, kind, K, M, R, lens, ids, n=3, pad=0, lead=0, seed=5, adapter_pad=0):
        self.kind, self.K, self.M, self.R, self.lens, self.ids, self.n = kind, K, M, R, list(lens), list(ids), n
        rng = np.random.default_rng(seed)
        self.T = int(sum(lens))
        self.a, self.a64 = encode(rng.standard_normal((n, R, K)) * K ** -0.5, kind)
        self.b, self.b64 = encode(rng.standard_normal((n, M, R)) * 0.1, kind)
        self.scale = rng.uniform(0.5, 2.0, n).astype(np.float32)
        f = lambda *s: rng.standard_normal(s).astype(np.float32)
        self.x, self.base, self.dy, self.dxb = f(self.T, K), f(self.T, M), f(self.T, M), f(self.T, K)
        self.start = starts(self.lens)
        self.pad, self.lead = pad, lead
        self.keep = []
        t = TYPES[kind]
        self.set = H.lora_set(self.adapters(self.a, t, adapter_pad), self.adapters(self.b, t, adapter_pad),
                              self.vector(self.scale, H.TYPE_F32), self.vector(self.start, H.TYPE_I32),
                              self.vector(np.array(self.ids, np.int32), H.TYPE_I32))

    def adapters(self, w, t, pad):
        n, r, c = w.shape
        base = np.zeros((n, r + (1 if pad else 0), c + pad), w.dtype)
        base[:, :r, :c] = w
        d = Dev(base)
        self.keep.append(d)
        es = w.dtype.itemsize
        return H.tensor(d.ptr, [c, r, n, 1], [es, es * base.shape[2], es * base[0].size, es * base.size], t)

    def vector(self, x, t):
        d, out = vec(x, t)
        self.keep.append(d)
        return out

    def mat(self, x):
        m = Mat(np.ascontiguousarray(x, np.float32), H.TYPE_F32, self.pad, self.lead)
        self.keep.append(m)
        return m

    def packed(self, x):
        m = Mat(np.ascontiguousarray(x, np.float32))
        self.keep.append(m)
        return m

    def requests(self):
        for q, i in enumerate(self.ids):
            if 0 <= i < self.n and self.lens[q]:
                yield i, slice(int(self.start[q]), int(self.start[q + 1]))

    def free(self):
        for k in self.keep:
            k.free()

    # ---- in 64 bits: results, and the same sums of magnitudes
    def forward(self, base):
        x, R = self.x.astype(np.float64), self.R
        h, y = np.zeros((self.T, R)), base.astype(np.float64).copy()
        hm, ym = np.zeros_like(h), np.abs(y)
        for i, r in self.requests():
            s = float(self.scale[i])
            h[r], hm[r] = x[r] @ self.a64[i].T, np.abs(x[r]) @ np.abs(self.a64[i]).T
            y[r] += s * h[r] @ self.b64[i].T
            ym[r] += s * hm[r] @ np.abs(self.b64[i]).T
        return h, hm, y, ym

    def backward(self, base, h):
        x, dy, h = self.x.astype(np.float64), self.dy.astype(np.float64), h.astype(np.float64)
        g, dx = np.zeros((self.T, self.R)), base.astype(np.float64).copy()
        gm, dxm = np.zeros_like(g), np.abs(dx)
        da, db = np.zeros_like(self.a64), np.zeros_like(self.b64)
        dam, dbm = np.zeros_like(da), np.zeros_like(db)
        for i, r in self.requests():
            s = float(self.scale[i])
            g[r], gm[r] = s * dy[r] @ self.b64[i], s * np.abs(dy[r]) @ np.abs(self.b64[i])
            dx[r] += g[r] @ self.a64[i]
            dxm[r] += gm[r] @ np.abs(self.a64[i])
            da[i] += g[r].T @ x[r]
            dam[i] += gm[r].T @ np.abs(x[r])
            db[i] += s * dy[r].T @ h[r]
            dbm[i] += s * np.abs(dy[r]).T @ np.abs(h[r])
        return (g, gm), (dx, dxm), (da, dam), (db, dbm)


def near(got, want, mags, n, what):
    bound = 8 * np.sqrt(n) * U32 * mags + 1e-30
    over = np.abs(got.astype(np.float64) - want) / bound
    assert np.all(over <= 1), f"{what}: {over.max():.2f} of the bound at {np.unravel_index(over.argmax(), over.shape)}"


def run_forward(p, use_base=True, in_place=False, stream=None):
    x, h = p.mat(p.x), p.packed(np.full((p.T, p.R), np.nan))
    base = p.mat(p.base) if use_base else None
    y = base if in_place else p.mat(np.full((p.T, p.M), np.nan))
    H.lora(p.set, x.t, base.t if base else None, h.t, y.t, stream)
    H.sync(stream)
    return h.read(), y.read()


def check_forward(p, **kw):
    h, y = run_forward(p, **kw)
    wh, hm, wy, ym = p.forward(p.base if kw.get("use_base", True) else np.zeros_like(p.base))
    near(h, wh, hm, p.K + 2, "h")
    near(y, wy, ym, p.K + p.R + 4, "y")
    p.free()


def run_backward(p, h, accumulate=False, use_base=True, in_place=False, use_dx=True, da0=None, db0=None, stream=None):
    x, hd, dy = p.mat(p.x), p.packed(h), p.mat(p.dy)
    g = p.packed(np.full((p.T, p.R), np.nan))
    base = p.mat(p.dxb) if use_base and use_dx else None
    dx = None if not use_dx else base if in_place else p.mat(np.full((p.T, p.K), np.nan))
    da, db = (p.packed(w.reshape(-1, w.shape[2])) for w in (da0, db0))
    view = lambda m, w: H.tensor(m.t.data, [w.shape[2], w.shape[1], w.shape[0], 1],
                                 [4, 4 * w.shape[2], 4 * w[0].size, 4 * w.size])
    H.lora_back(p.set, x.t, hd.t, dy.t, g.t, base.t if base else None, dx.t if dx else None, view(da, da0), view(db, db0),
                accumulate, stream)
    H.sync(stream)
    return g.read(), dx.read() if dx else None, da.read().reshape(da0.shape), db.read().reshape(db0.shape)


def check_backward(p, accumulate=False, use_base=True, **kw):
    rng = np.random.default_rng(9)
    h = rng.standard_normal((p.T, p.R)).astype(np.float32)
    da0, db0 = (rng.standard_normal(w.shape).astype(np.float32) for w in (p.a64, p.b64))
    g, dx, da, db = run_backward(p, h, accumulate, use_base, da0=da0, db0=db0, **kw)
    (wg, gm), (wdx, dxm), (wda, dam), (wdb, dbm) = p.backward(p.dxb if use_base else np.zeros_like(p.dxb), h)
    if accumulate:
        wda, dam, wdb, dbm = wda + da0, dam + np.abs(da0), wdb + db0, dbm + np.abs(db0)
    near(g, wg, gm, p.M + 3, "g")
    if dx is not None:
        near(dx, wdx, dxm, p.M + p.R + 5, "dx")
    near(da, wda, dam, p.M + p.T + 5, "da")
    near(db, wdb, dbm, p.T + 5, "db")
    p.free()


SHAPES = [  # K, M, R, lens, ids
    (64, 48, 8, [1], [1]),
    (1, 1, 1, [1], [0]),
    (3, 5, 2, [2, 1], [2, 0]),
    (100, 77, 16, [1, 1, 1, 1, 1], [0, 1, 2, 1, -1]),
    (257, 130, 17, [3, 0, 19, 16, 1], [1, 0, -1, 2, 0]),
    (768, 288, 4, [33], [2]),
    (1000, 777, 24, [15, 17, 31, 64], [0, 0, 2, 1]),
    (512, 1030, 64, [40, 7], [1, 2]),
    (130, 515, 65, [18, 5], [2, 0]),
    (96, 64, 128, [16, 1, 2], [0, 1, 3]),      # 3: no such adapter
    (70, 40, 256, [5, 4], [1, -7]),
]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward(hip, kind, shape):
    announce(f"lora forward {kind} {shape}")
    check_forward(Problem(kind, *shape))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_backward(hip, kind, shape):
    announce(f"lora backward {kind} {shape}")
    check_backward(Problem(kind, *shape))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("pad,lead,adapter_pad", [(1, 1, 1), (3, 2, 5), (4, 4, 8), (129, 3, 0)])
def test_strides(hip, kind, pad, lead, adapter_pad):
    """Rows apart by any number of elements and from any element on; what lies between stays."""
    announce(f"lora strides {kind} {pad} {lead} {adapter_pad}")
    shape = (203, 150, 20, [1, 18, 2], [2, 0, 1])
    check_forward(Problem(kind, *shape, pad=pad, lead=lead, adapter_pad=adapter_pad))
    check_backward(Problem(kind, *shape, pad=pad, lead=lead, adapter_pad=adapter_pad))


@pytest.mark.parametrize("use_base,in_place", [(False, False), (True, True)])
def test_base(hip, use_base, in_place):
    announce(f"lora base {use_base} {in_place}")
    shape = (130, 94, 12, [5, 1, 17], [0, -1, 1])
    check_forward(Problem("f16", *shape, pad=2), use_base=use_base, in_place=in_place)
    check_backward(Problem("f16", *shape, pad=2), use_base=use_base, in_place=in_place)


def test_back_without_dx_and_accumulated(hip):
    announce("lora backward without dx, accumulated")
    check_backward(Problem("f32", 300, 200, 16, [50, 3], [0, 2]), accumulate=True, use_dx=False)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_long_axis_and_few_tokens(hip, kind):
    """One token over a long axis: its sums meet in parts."""
    announce(f"lora long axis {kind}")
    for K, M, R, lens, ids in [(14336, 200, 64, [1], [1]), (8195, 64, 5, [1, 2], [0, 2]), (4099, 4099, 100, [3], [0])]:
        check_forward(Problem(kind, K, M, R, lens, ids))
        check_backward(Problem(kind, K, M, R, lens, ids))


def test_many_requests(hip):
    """More requests than a wave has lanes, most of one token, some of none."""
    announce("lora many requests")
    rng = np.random.default_rng(2)
    lens = [int(v) for v in rng.choice([0, 1, 1, 1, 2, 16, 17, 40], 200)]
    ids = [int(v) for v in rng.integers(-1, 6, 200)]
    check_forward(Problem("f16", 160, 200, 16, lens, ids, n=5))
    check_backward(Problem("f16", 160, 200, 16, lens, ids, n=5))


def test_more_requests_than_a_workgroup_has_lanes(hip):
    announce("lora 1500 requests")
    rng = np.random.default_rng(3)
    lens = [int(v) for v in rng.choice([0, 1, 1, 1, 2, 18], 1500)]
    ids = [int(v) for v in rng.integers(-1, 6, 1500)]
    check_forward(Problem("f16", 60, 90, 8, lens, ids, n=5))
    check_backward(Problem("f16", 60, 90, 8, lens, ids, n=5))
    check_forward(Problem("f32", 2100, 1030, 40, [0] * 300 + [3, 0, 1], [0] * 301 + [1, 2]))


def test_many_tokens(hip):
    announce("lora many tokens")
    check_forward(Problem("f32", 260, 520, 32, [3000, 1, 1100], [1, 0, 2]))
    check_backward(Problem("f32", 260, 520, 32, [3000, 1, 1100], [1, 0, 2]))


@pytest.mark.parametrize("kind", list(TYPES))
def test_single_tokens_of_high_ranks_over_a_long_axis(hip, kind):
    announce(f"lora single tokens, high ranks {kind}")
    check_forward(Problem(kind, 8200, 300, 200, [1, 1, 1, 2], [0, 2, -1, 1]))
    check_forward(Problem(kind, 6000, 70, 67, [1], [1], pad=1, lead=1, adapter_pad=1))


@pytest.mark.parametrize("kind", list(TYPES))
def test_gradients_of_few_tokens_over_many_columns(hip, kind):
    """g's sums are long and its tiles few: they meet in parts."""
    announce(f"lora gradients, few tokens, many columns {kind}")
    check_backward(Problem(kind, 300, 2100, 20, [40, 3, 1], [1, 0, -1]), accumulate=True)
    check_backward(Problem(kind, 70, 1537, 16, [17], [2], pad=1))
    check_backward(Problem(kind, 1100, 4111, 3, [1, 30], [0, 0]), in_place=True)


@pytest.mark.parametrize("use_base,in_place", [(True, False), (False, False), (True, True)])
def test_many_tokens_without_an_adapter(hip, use_base, in_place):
    """Their base is passed on, many columns of it to a workgroup."""
    announce(f"lora many tokens without an adapter, base {use_base}, in place {in_place}")
    check_forward(Problem("f16", 24, 3300, 8, [4200, 40], [-1, 1], n=2), use_base=use_base, in_place=in_place)


@pytest.mark.parametrize("accumulate", [False, True])
def test_gradients_of_one_small_adapter_over_many_tokens(hip, accumulate):
    """Few columns and thousands of tokens: the gradients' tokens are split, and the parts joined."""
    announce(f"lora one adapter, many tokens, accumulate {accumulate}")
    check_backward(Problem("bf16", 70, 40, 6, [4500, 1, 1710], [0, 0, 0], n=1), accumulate=accumulate)
    check_backward(Problem("f32", 35, 33, 17, [4097], [0], n=1), accumulate=accumulate, use_dx=False)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_values_that_are_not_finite_stay_with_their_token(hip, bad):
    """... and with their adapter: a token without one only passes its base on, and a neighbour in
    the same tile, or a request of another adapter, sees nothing of them."""
    announce(f"lora not finite {bad}")
    p = Problem("f32", 90, 70, 10, [3, 4, 2], [0, 1, -1])
    p.x[1] = bad          # request 0
    p.x[8] = bad          # a token without an adapter
    h, y = run_forward(p)
    assert not np.isfinite(h[1]).any() and not np.isfinite(y[1]).any()
    p.x[1], p.x[8] = 0, 0
    wh, hm, wy, ym = p.forward(p.base)
    rest = [0, 2, 3, 4, 5, 6, 7, 8]
    near(h[rest], wh[rest], hm[rest], p.K + 2, "h")
    near(y[rest], wy[rest], ym[rest], p.K + p.R + 4, "y")
    assert np.array_equal(y[7:], p.base[7:]) and not h[7:].any()
    p.free()

    p = Problem("f32", 90, 70, 10, [3, 4, 2], [0, 1, -1])
    p.dy[8], p.x[8] = bad, bad
    p.x[0] = bad          # dA of adapter 0 alone
    hh = np.random.default_rng(4).standard_normal((p.T, p.R)).astype(np.float32)
    hh[8] = bad
    g, dx, da, db = run_backward(p, hh, da0=np.zeros_like(p.a, dtype=np.float32), db0=np.zeros_like(p.b, dtype=np.float32))
    p.x[0], p.x[8], p.dy[8], hh[8] = 0, 0, 0, 0
    (wg, gm), (wdx, dxm), (wda, dam), (wdb, dbm) = p.backward(p.dxb, hh)
    assert not np.isfinite(da[0]).any()
    near(da[1:], wda[1:], dam[1:], p.M + p.T + 5, "da")
    near(db, wdb, dbm, p.T + 5, "db")
    near(dx, wdx, dxm, p.M + p.R + 5, "dx")
    assert np.array_equal(dx[7:], p.dxb[7:]) and not da[2].any()
    p.free()


@pytest.mark.parametrize("start", [[0, 100, 7], [-5, 3, 2000000000], [7, 3, 0], [2147483647, -2147483648, 5]])
def test_wrong_starts_stay_inside_the_tensors(hip, start):
    announce(f"lora wrong starts {start}")
    p = Problem("f16", 40, 30, 6, [4, 3], [0, 1], pad=3, lead=1)
    d, t = vec(np.array(start, np.int32), H.TYPE_I32)
    p.keep.append(d)
    p.set.start = t
    run_forward(p)  # Mat.read() checks what lies around the rows
    run_backward(p, np.zeros((p.T, p.R), np.float32), da0=np.zeros(p.a.shape, np.float32), db0=np.zeros(p.b.shape, np.float32))
    p.free()


def test_gradients_against_differences(hip):
    """L = sum c y is linear in x, in A and in B by itself, so a difference over a step of any
    size is its derivative, but for the rounding of the two forward passes."""
    announce("lora differences")
    rng = np.random.default_rng(6)
    shape = ("f32", 120, 90, 12, [5, 1, 20], [0, 2, 1])

    def loss(**change):
        p = Problem(*shape)
        for k, v in change.items():
            setattr(p, k, v)
        q = Problem(*shape)  # the same sizes; its adapters replaced
        for w, name in ((p.a, "a"), (p.b, "b")):
            setattr(q.set, name, q.adapters(np.ascontiguousarray(w, np.float32), H.TYPE_F32, 0))
        q.x = p.x
        _, y = run_forward(q)
        out = float((p.dy.astype(np.float64) * y).sum())
        mag = float((np.abs(p.dy).astype(np.float64) * np.abs(y)).sum())
        p.free()
        q.free()
        return out, mag

    p = Problem(*shape)
    h, _ = run_forward(p)
    _, dx, da, db = run_backward(p, h, use_base=False, da0=np.zeros(p.a.shape, np.float32), db0=np.zeros(p.b.shape, np.float32))
    for name, grad in (("x", dx), ("a", da), ("b", db)):
        step = rng.standard_normal(grad.shape).astype(np.float32)
        at = getattr(p, name)
        (hi, m1), (lo, m2) = loss(**{name: at + step}), loss(**{name: at - step})
        want = float((grad.astype(np.float64) * step).sum())
        # each y is off by at most 8 sqrt(K + R) 2^-24 of its magnitudes, taken as 30 times the values here
        assert abs((hi - lo) / 2 - want) <= 30 * 8 * np.sqrt(p.K + p.R) * U32 * (m1 + m2), name
    p.free()


def test_same_bits_on_streams_and_under_capture(hip):
    """Other streams and replays of a captured graph give the first call's bits, also where
    the sums meet in the stream's workspace, with eager calls in between."""
    announce("lora streams and capture")
    rt = runtime()
    for shape in [("f16", 4096, 300, 16, [1, 1, 1], [0, 1, 2]), ("f32", 300, 260, 20, [100, 3], [0, 1])]:
        p = Problem(*shape)
        want = run_forward(p)
        s = Stream()
        x, base = p.mat(p.x), p.mat(p.base)
        h, y = p.packed(np.zeros((p.T, p.R))), p.mat(np.zeros((p.T, p.M)))
        H.lora(p.set, x.t, base.t, h.t, y.t, s.handle)
        H.sync(s.handle)
        assert np.array_equal(h.read(), want[0]) and np.array_equal(y.read(), want[1])
        graph, gexec = C.c_void_p(), C.c_void_p()
        assert rt.hipStreamBeginCapture(C.c_void_p(s.handle), 0) == 0
        try:
            H.lora(p.set, x.t, base.t, h.t, y.t, s.handle)
        finally:
            rc = rt.hipStreamEndCapture(C.c_void_p(s.handle), C.byref(graph))
        assert rc == 0 and rt.hipGraphInstantiate(C.byref(gexec), graph, None, None, 0) == 0
        for _ in range(3):
            H.fill_f32(y.t.data, 0.0, p.T * p.M)
            H.sync()
            assert rt.hipGraphLaunch(gexec, C.c_void_p(s.handle)) == 0
            H.sync(s.handle)
            assert np.array_equal(y.read(), want[1])
            got = run_forward(p)
            assert np.array_equal(got[1], want[1])
        rt.hipGraphExecDestroy(gexec)
        rt.hipGraphDestroy(graph)
        s.close()
        p.free()
