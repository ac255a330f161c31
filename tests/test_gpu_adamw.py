"""AdamW over many tensors (trc_hip_adamw_*): against 64 bits, against the reference's own
trajectories, and the 8-bit moments against their definition.

Tolerance: one step rounds m and v three times each, and the update m / (sqrt(v) / root + eps)
* rate some eight more, each by 2^-24 of its value, where m's two terms may cancel:
m within 4 * 2^-24 (|b1 m| + |c1 g|), v within 4 * 2^-24 v, p within 2^-24 |p| for each of its two
roundings, its decay's factor, and 16 * 2^-24 of the update's magnitudes."""
import numpy as np
import pytest

from conftest import GOLDEN, announce
from gpu_util import Dev, Stream
from traincpp_amd import hip as H
from tuning_util import TYPES, U32, encode

pytestmark = pytest.mark.gpu

HYPER = dict(lr=1e-2, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1)
M_UNIT, U_UNIT = np.float32(1 / 127 ** 2), np.float32(1 / 255 ** 2)


class Tensors:
    """Tensors with their gradients and moments in one buffer each, `lead` elements in."""

    def __init__(self, sizes, bits=32, kind="f32", lead=0, seed=1, decay=None):
        rng = np.random.default_rng(seed)
        self.sizes, self.bits, self.kind, self.lead = list(sizes), bits, kind, lead
        self.decay = decay or [1.0] * len(self.sizes)
        self.p = [rng.standard_normal(n).astype(np.float32) for n in sizes]
        self.g, self.g64 = zip(*[encode(rng.standard_normal(n) * 0.1, kind) for n in sizes]) if sizes else ((), ())
        self.blocks = [-(-n // H.ADAMW_BLOCK) for n in sizes]
        self.bufs = {"param": self.up(self.p), "grad": self.up(self.g)}
        dt = (np.float32, np.float32) if bits == 32 else (np.int8, np.uint8)
        for k, d in zip(("m", "v"), dt):
            self.bufs[k] = self.up([np.zeros(n, d) for n in sizes])
            self.bufs[k + "_out"] = self.up([np.full(n, np.nan, np.float32) for n in sizes])
            if bits == 8:
                self.bufs[k + "_scale"] = self.up([np.zeros(n, np.float32) for n in self.blocks])
        self.plan = H.AdamW([dict(n=n, decay=self.decay[i], grad_type=TYPES[kind],
                                  **{k: self.ptr(k, i) for k in self.bufs}) for i, n in enumerate(self.sizes)], bits)

    def up(self, arrays):
        """[lead marks][array][one mark] for each array, one after the other."""
        out, at = [], []
        n = 0
        for a in arrays:
            mark = np.full(self.lead + 1, 85, a.dtype)
            at.append(n + self.lead)
            out += [mark[:self.lead], a, mark[:1]]
            n += self.lead + a.size + 1
        base = np.concatenate(out) if out else np.zeros(1, np.float32)
        return Dev(base), at, [a.size for a in arrays]

    def ptr(self, k, i):
        d, at, _ = self.bufs[k]
        return d.ptr + at[i] * d.base.itemsize

    def read(self, k):
        d, at, n = self.bufs[k]
        base = d.read()
        keep = np.ones(base.shape, bool)
        for a, c in zip(at, n):
            keep[a:a + c] = False
        if n:
            assert np.all(base[keep] == 85), f"{k}: elements outside the tensors were written"
        return [base[a:a + c].copy() for a, c in zip(at, n)]

    def write(self, k, arrays):
        d, at, n = self.bufs[k]
        for a, c, x in zip(at, n, arrays):
            d.base[a:a + c] = x
        d.buf.upload(d.base)

    def free(self):
        self.plan.destroy()
        for d, _, _ in self.bufs.values():
            d.free()


def expected(p, g, m, v, step, decay, lr, beta1, beta2, eps, weight_decay, grad_scale=1.0):
    """The new p, m, v in 64 bits, and the bounds of the module's comment."""
    p, m, v, g = (np.asarray(q, np.float64) for q in (p, m, v, g))
    g = g * grad_scale
    mb = 4 * U32 * (beta1 * np.abs(m) + (1 - beta1) * np.abs(g))
    m, v = beta1 * m + (1 - beta1) * g, beta2 * v + (1 - beta2) * g * g
    with np.errstate(all="ignore"):
        div = np.sqrt(v / (1 - beta2 ** step)) + eps
        rate = lr / (1 - beta1 ** step)
        new = p - lr * weight_decay * decay * p - rate * m / div
        pb = 4 * U32 * (np.abs(p) + np.abs(new)) + rate * (16 * U32 * np.abs(m) + mb) / div
    return (new, pb), (m, mb + 1e-45), (v, 4 * U32 * v + 1e-44)


def near(got, want, what):
    w, bound = want
    over = np.abs(got.astype(np.float64) - w) / (bound + 1e-45)
    assert got.size == 0 or np.all(over <= 1), f"{what}: {over.max()} of the bound"


SIZES = [[1], [3, 1, 4, 0, 5], [255, 256, 257], [4095, 4096, 4097, 1], [100003, 7, 8192 * 3], [64] * 300]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("lead", [0, 1, 3])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
def test_32_bits(hip, kind, lead, sizes):
    announce(f"adamw 32 {kind} lead={lead} {sizes[:5]}")
    decay = [1.0 if i % 3 else 0.0 for i in range(len(sizes))]
    t = Tensors(sizes, 32, kind, lead, decay=decay)
    p, m, v = t.p, [np.zeros(n) for n in sizes], [np.zeros(n) for n in sizes]
    for step in (1, 2, 100):
        t.plan.step(step=step, grad_scale=0.5 if step == 2 else 1.0, **HYPER)
        H.sync()
        got = [t.read(k) for k in ("param", "m", "v")]
        for i in range(len(sizes)):
            want = expected(p[i], t.g64[i], m[i], v[i], step, decay[i], grad_scale=0.5 if step == 2 else 1.0, **HYPER)
            for name, q, w in zip("pmv", got, want):
                near(q[i], w, f"{name} of tensor {i}, step {step}")
        p, m, v = got
    t.plan.moments()
    H.sync()
    assert all(np.array_equal(a, b) for k, q in (("m_out", m), ("v_out", v)) for a, b in zip(t.read(k), q))
    t.free()


def inverse(s):
    with np.errstate(all="ignore"):
        return np.where(s >= np.float32(2.0 ** -126), np.float32(1) / s, np.float32(0)).astype(np.float32)


def unpack(code, scale, unit, n):
    c = np.zeros(-(-n // 256) * 256, np.float32)
    c[:n] = code
    c = c.reshape(-1, 256)
    return ((np.abs(c) * c * scale[:, None]) * unit).reshape(-1)[:n].astype(np.float32)


def pack(x, full, lowest):
    n = x.size
    b = np.zeros(-(-n // 256) * 256, np.float32)
    b[:n] = x
    b = b.reshape(-1, 256)
    scale = np.abs(b).max(1)
    inv = inverse(scale)
    ratio = np.abs(b) * inv[:, None]
    c = np.rint(np.sqrt(ratio) * np.float32(full))
    if lowest:
        c = np.where(ratio > 0, np.maximum(c, 1), c)
    return np.where(b < 0, -c, c).reshape(-1)[:n], np.where(inv > 0, scale, np.float32(0))


def step8(p, g, m8, ms, u8, us, step, decay, lr, beta1, beta2, eps, weight_decay):
    """One step with every operation rounded to 32 bits on its own, in the documented order."""
    f = np.float32
    g = g.astype(f)
    m, u = unpack(m8, ms, M_UNIT, p.size), unpack(u8, us, U_UNIT, p.size)
    m = m * f(beta1) + g * f(1 - beta1)
    v = (u * u) * f(beta2) + (g * g) * f(1 - beta2)
    u = np.sqrt(v)
    with np.errstate(all="ignore"):
        p = p * f(1 - lr * weight_decay * decay)
        p = p - (m / (u * f(1 / np.sqrt(1 - beta2 ** step)) + f(eps))) * f(lr / (1 - beta1 ** step))
    return (p, *pack(m, 127, False), *pack(u, 255, True), m, u)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("lead", [0, 1, 2])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
def test_8_bits(hip, kind, lead, sizes):
    """Codes, scales and parameters, bit for bit, over several steps; gradients of widely
    different sizes in a block."""
    announce(f"adamw 8 {kind} lead={lead} {sizes[:5]}")
    decay = [0.0 if i % 3 else 1.0 for i in range(len(sizes))]
    t = Tensors(sizes, 8, kind, lead, decay=decay)
    rng = np.random.default_rng(7)
    state = [(t.p[i], np.zeros(n), np.zeros(t.blocks[i], np.float32), np.zeros(n), np.zeros(t.blocks[i], np.float32))
             for i, n in enumerate(sizes)]
    for step in (1, 2, 50):
        g, g64 = zip(*[encode(rng.standard_normal(n) * 10.0 ** rng.uniform(-4, 1, n), kind) for n in sizes])
        t.write("grad", g)
        t.plan.step(step=step, **HYPER)
        t.plan.moments()
        H.sync()
        p, m8, ms, u8, us, mo, vo = (t.read(k) for k in ("param", "m", "m_scale", "v", "v_scale", "m_out", "v_out"))
        for i, n in enumerate(sizes):
            if n == 0:
                continue
            p0, a, b, c, d = state[i]
            w = step8(p0, g64[i], a, b, c, d, step, decay[i], **HYPER)
            assert np.array_equal(m8[i], w[1]) and np.array_equal(ms[i], w[2]), f"m of tensor {i}, step {step}"
            assert np.array_equal(u8[i], w[3]) and np.array_equal(us[i], w[4]), f"v of tensor {i}, step {step}"
            assert np.array_equal(p[i], w[0]), f"p of tensor {i}, step {step}"
            assert np.array_equal(mo[i], unpack(w[1], w[2], M_UNIT, n))
            u = unpack(w[3], w[4], U_UNIT, n)
            assert np.array_equal(vo[i], u * u)
            # what the codes stand for: within half a step of the code, and never 0 under a v above it
            assert np.all(u8[i][w[6] > 0] > 0)
            unit = np.repeat(ms[i], 256)[:n]
            assert np.all(np.abs(mo[i] - w[5]) <= unit * (np.abs(m8[i].astype(np.float64)) + 0.5) / 127 ** 2 + 1e-30)
            state[i] = (p[i], m8[i], ms[i], u8[i], us[i])
    t.free()


def test_8_bit_blocks_of_zeros_and_of_tiny_values(hip):
    announce("adamw 8 zeros and tiny values")
    t = Tensors([512, 300], 8)
    g = [np.zeros(512, np.float32), np.full(300, 1e-38, np.float32)]
    g[0][300] = 1e-42
    t.write("grad", g)
    t.plan.step(step=1, **HYPER)
    H.sync()
    p = t.read("param")
    assert np.all(np.isfinite(p[0])) and np.all(np.isfinite(p[1]))
    assert not t.read("m")[0].any() and not t.read("m_scale")[0].any() and not t.read("v_scale")[0].any()
    assert np.array_equal(p[0][:256], (t.p[0] * np.float32(1 - HYPER["lr"] * HYPER["weight_decay"]))[:256])
    t.free()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_gradients_that_are_not_finite(hip, bits, bad):
    """One bad gradient: its own element with 32 bits, with 8 its block's moments from then on;
    every other block and tensor is as without it."""
    announce(f"adamw not finite {bits} {bad}")
    a, b = Tensors([700, 40], bits), Tensors([700, 40], bits)
    g = [x.copy() for x in a.g]
    g[0][300] = bad
    b.write("grad", g)
    for t in (a, b):
        t.plan.step(step=1, **HYPER)
        t.plan.moments()
    H.sync()
    ps, ms = [t.read("param") for t in (a, b)], [t.read("m_out") for t in (a, b)]
    assert not np.isfinite(ps[1][0][300])
    other = np.arange(700) != 300
    assert np.array_equal(ps[0][0][other], ps[1][0][other]) and np.array_equal(ps[0][1], ps[1][1])
    block = other if bits == 32 else np.arange(700) // 256 != 1
    assert np.array_equal(ms[0][0][block], ms[1][0][block]) and not np.isfinite(ms[1][0][~block]).any()
    a.free()
    b.free()


@pytest.mark.parametrize("name", ["optim_adamw_basic", "optim_adamw_nowd"])
def test_reference_trajectories(hip, name):
    """The reference's own AdamW trajectories, all parameters in one plan. Each of six steps adds
    the roundings of one step (2^-24 of values up to 4, some 30 of them)."""
    announce(f"adamw {name}")
    d = GOLDEN / "reference_suite"
    meta = dict(l.split(None, 1) for l in (d / f"{name}_meta.txt").read_text().splitlines() if l.strip())
    init = [np.load(d / f"{name}_p{i}_init.npy") for i in range(int(meta["nparams"]))]
    grads = [np.load(d / f"{name}_p{i}_grads.npy") for i in range(len(init))]
    traj = [np.load(d / f"{name}_p{i}_traj.npy") for i in range(len(init))]
    t = Tensors([x.size for x in init])
    t.write("param", [x.ravel() for x in init])
    for step in range(int(meta["steps"])):
        t.write("grad", [g[step].ravel() for g in grads])
        t.plan.step(lr=float(meta["lr"]), step=step + 1, beta1=float(meta["beta1"]), beta2=float(meta["beta2"]),
                    eps=float(meta["eps"]), weight_decay=float(meta["weight_decay"]))
        H.sync()
        for i, p in enumerate(t.read("param")):
            assert np.abs(p - traj[i][step + 1].ravel()).max() <= (step + 1) * 30 * 4 * U32
    t.free()


def test_8_bits_follow_32(hip):
    """Two hundred steps down a quadratic bowl with noisy gradients: the 8-bit moments get as far."""
    announce("adamw 8 bits against 32")
    n = 2000
    rng = np.random.default_rng(3)
    goal = rng.standard_normal(n).astype(np.float32)
    left = {}
    for bits in (32, 8):
        noise = np.random.default_rng(4)
        t = Tensors([n], bits, seed=11)
        p = t.p[0]
        for step in range(1, 201):
            t.write("grad", [((p - goal) * np.linspace(0.01, 3, n) + noise.standard_normal(n) * 1e-3).astype(np.float32)])
            t.plan.step(lr=0.05, step=step, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0)
            H.sync()
            p = t.read("param")[0]
        left[bits] = float(np.abs(p - goal).mean())
        t.free()
    start = float(np.abs(np.random.default_rng(11).standard_normal(n).astype(np.float32) - goal).mean())
    assert left[32] < 0.05 * start and left[8] < 0.05 * start, (left, start)


def test_plans_without_work(hip):
    announce("adamw empty plans")
    for sizes in ([], [0], [0, 0]):
        t = Tensors(sizes)
        t.plan.step(step=1, **HYPER)
        t.plan.moments()
        H.sync()
        t.free()


def test_streams(hip):
    announce("adamw streams")
    a, b = Tensors([5000, 33], 8), Tensors([5000, 33], 8)
    s = Stream()
    for step in (1, 2, 3):
        a.plan.step(step=step, **HYPER)
        b.plan.step(step=step, stream=s.handle, **HYPER)
    H.sync()
    H.sync(s.handle)
    for k in ("param", "m", "v", "m_scale", "v_scale"):
        assert all(np.array_equal(x, y) for x, y in zip(a.read(k), b.read(k)))
    s.close()
    a.free()
    b.free()


def test_moments_need_their_destinations(hip):
    announce("adamw moments refused")
    t = Tensors([10])
    plan = H.AdamW([dict(param=t.ptr("param", 0), grad=t.ptr("grad", 0), m=t.ptr("m", 0), v=t.ptr("v", 0), n=10)])
    with pytest.raises(H.HipError) as e:
        plan.moments()
    assert e.value.code == H.E_INVALID
    plan.destroy()
    t.free()
