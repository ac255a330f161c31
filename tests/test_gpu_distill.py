"""The distillation loss (trc_hip_distill_loss) and its gradient against 64 bits.

Tolerance, with u = 2^-24. A row's sums are of V positive terms: each an exponential whose argument is rounded (its magnitude, up
to the logits' spread over tau, times u) and exp2 itself (2 u), added in chains of n a thread and a tree:
e_s = (spread / min(tau, 1) + 8 sqrt(V) + 8) u relative (squared exponentials twice that of the root's). KL and CE add e_s for the logarithm of a
sum; the rest of them is in 64 bits, rounded once. A gradient's exponential has the same argument error, its sum e_s, and its
factors 8 u; the teacher's probabilities (spread of the teacher / tau + 8) u. 16 bits round it once more."""
import ctypes as C

import numpy as np
import pytest

from conftest import announce
from gpu_util import Stream, runtime
from traincpp_amd import hip as H
from tuning_util import TYPES, U32, Mat, decode, encode, vec

pytestmark = pytest.mark.gpu

HALF = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


class Problem:
    def __init__(self, kind, V, T, top, tau=2.0, alpha=0.5, seed=3, tkind="f32", pad=0, lead=0, skip=0.25):
        rng = np.random.default_rng(seed)
        self.kind, self.V, self.T, self.top, self.tau, self.alpha = kind, V, T, top, np.float32(tau), np.float32(alpha)
        self.tkind, self.pad, self.lead = tkind, pad, lead
        self.logits, self.l64 = encode(rng.standard_normal((T, V)) * 3, kind)
        self.teacher, self.z64 = encode(rng.standard_normal((T, top)) * 2 + 5, tkind)
        self.ids = np.stack([rng.permutation(V)[:top] if V >= top else rng.integers(0, V, top) for _ in range(T)]).astype(np.int32)
        self.labels = rng.integers(0, V, T).astype(np.int32)
        for t in range(0, T, 3):
            self.labels[t] = self.ids[t, t % top]  # a label among the teacher's tokens
        self.labels[rng.random(T) < skip] = -1
        self.dloss = np.array([0.7], np.float32)

    def views(self, in_place=False):
        keep = []

        def v(x, kind=H.TYPE_F32):
            d, t = vec(x, kind)
            keep.append(d)
            return d, t

        m = Mat(self.logits, TYPES[self.kind], self.pad, self.lead)
        d = m if in_place else Mat(np.zeros_like(self.logits), TYPES[self.kind], self.pad, self.lead)
        ids, teacher = Mat(self.ids, H.TYPE_I32), Mat(self.teacher, TYPES[self.tkind])
        stats = Mat(np.full((self.T, 5), np.nan, np.float32))
        keep += [m, ids, teacher, stats] + ([] if in_place else [d])
        _, labels = v(self.labels, H.TYPE_I32)
        loss, loss_t = v(np.full(4, np.nan, np.float32))
        _, dloss = v(self.dloss)
        fwd = (m.t, labels, ids.t, teacher.t, self.tau, self.alpha, stats.t, loss_t)
        back = (m.t, labels, ids.t, teacher.t, stats.t, loss_t, dloss, self.tau, self.alpha, d.t)
        return fwd, back, loss, d, stats, keep

    def run(self, stream=None, in_place=False):
        fwd, back, loss, d, stats, keep = self.views(in_place)
        H.distill_loss(*fwd, stream)
        H.distill_loss_back(*back, stream)
        H.sync(stream)
        out = loss.read(), d.read()
        stats.read()
        for k in keep:
            k.free()
        return out

    def want(self):
        tau, alpha = float(self.tau), float(self.alpha)
        d = np.zeros_like(self.l64)
        kl = ce = 0.0
        n = int((self.labels >= 0).sum())
        with np.errstate(all="ignore"):
            for t in np.nonzero(self.labels >= 0)[0]:
                l, y = self.l64[t], self.labels[t]
                if alpha > 0:
                    ok = (self.ids[t] >= 0) & (self.ids[t] < self.V)
                    ids, z = self.ids[t][ok], self.z64[t][ok] / tau
                    if len(ids):
                        x = l / tau
                        logq = x - x.max() - np.log(np.exp(x - x.max()).sum())
                        logp = z - z.max() - np.log(np.exp(z - z.max()).sum())
                        p = np.exp(logp)
                        kl += np.where(p > 0, p * (logp - logq[ids]), 0).sum()
                        g = np.exp(logq)
                        np.add.at(g, ids, -p)
                        d[t] += alpha * tau * g
                if alpha < 1:
                    logr = l - l.max() - np.log(np.exp(l - l.max()).sum())
                    ce -= logr[y] if y < self.V else np.nan
                    g = np.exp(logr)
                    if y < self.V:
                        g[y] -= 1
                    d[t] += (1 - alpha) * g
            if n:
                kl, ce, d = kl / n, ce / n, d * (float(self.dloss[0]) / n)
        return np.array([alpha * tau * tau * kl + (1 - alpha) * ce, kl, ce, n]), d


def check(p, got=None, **kw):
    loss, d = got if got is not None else p.run(**kw)
    wl, wd = p.want()
    tau, alpha, n = float(p.tau), float(p.alpha), max(wl[3], 1)
    spread, zs = np.ptp(p.l64), np.ptp(p.z64)
    e_s = 2 * (spread / min(tau, 1) + 8 * np.sqrt(p.V) + 8) * U32
    assert loss[3] == wl[3]
    for i in (1, 2):
        assert abs(loss[i] - wl[i]) <= e_s + 2 * U32 * abs(wl[i]), (i, loss, wl)
    assert abs(loss[0] - wl[0]) <= e_s * (alpha * tau * tau + 1 - alpha) + 2 * U32 * abs(wl[0])
    # what the terms of a gradient can weigh: probabilities, and the entries' and the label's
    mag = np.zeros_like(wd)
    for t in np.nonzero(p.labels >= 0)[0]:
        for x, w in ((p.l64[t] / tau, alpha * tau), (p.l64[t], 1 - alpha)):
            mag[t] += w * np.exp(x - x.max()) / np.exp(x - x.max()).sum()
        ok = (p.ids[t] >= 0) & (p.ids[t] < p.V)
        np.add.at(mag[t], p.ids[t][ok], alpha * tau)  # (a probability, 1 at most)
        if p.labels[t] < p.V:
            mag[t, p.labels[t]] += 1 - alpha
    mag *= abs(float(p.dloss[0])) / n
    got = decode(d, p.kind)
    err = mag * (2 * e_s + (zs / tau + 16 + p.top) * U32)
    bound = err + HALF[p.kind] * (np.abs(wd) + err) + (2.0 ** -25 if p.kind == "f16" else 1e-36)
    over = np.abs(got - wd) / bound
    assert over.max() <= 1, f"dlogits: {over.max()} of the bound at {np.unravel_index(over.argmax(), over.shape)}"
    assert not got[p.labels < 0].any()


MIXES = [(1.0, 0.5), (2.0, 0.9), (2.0, 1.0), (4.0, 0.3), (1.5, 0.0), (0.5, 0.7), (1.0, 1.0)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("V,T,top", [(1, 2, 1), (2, 3, 2), (7, 30, 4), (1000, 40, 64), (4099, 9, 20), (8192, 5, 1), (32000, 17, 64),
                                     (131071, 5, 20), (333, 700, 3), (2500, 6, 1024)])
def test_loss_and_gradient(hip, kind, V, T, top):
    announce(f"distill {kind} V={V} T={T} top={top}")
    for i, (tau, alpha) in enumerate(MIXES):
        if V * T < 1 << 18 or i % 3 == 0:
            check(Problem(kind, V, T, top, tau, alpha, tkind=list(TYPES)[(i + V) % 3], seed=i))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("pad,lead", [(1, 1), (3, 5), (8, 8)])
def test_strided_rows(hip, kind, pad, lead):
    announce(f"distill strides {kind} {pad} {lead}")
    for tau, alpha in ((2.0, 0.5), (3.0, 0.5), (1.0, 1.0)):
        check(Problem(kind, 8209, 9, 12, tau, alpha, pad=pad, lead=lead))
        check(Problem(kind, 515, 9, 12, tau, alpha, pad=pad, lead=lead), in_place=True)


@pytest.mark.parametrize("V", [700, 70000])
def test_in_place(hip, V):
    """The gradient over the logits themselves, whole rows and rows in parts: the same bits."""
    announce(f"distill in place V={V}")
    for kind in TYPES:
        p = Problem(kind, V, 7, 40, 2.0, 0.5)
        p.ids[:, 1] = p.ids[:, 0]
        a, b = p.run(), p.run(in_place=True)
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("V,top", [(600, 1024), (40000, 1024), (40000, 300), (70000, 33)])
def test_many_repeated_entries(hip, kind, V, top):
    """All of a row's entries one token, pairs, runs, tokens that differ by powers of two, the label among them or not."""
    announce(f"distill many repeated {kind} V={V} top={top}")
    for alpha in (1.0, 0.6):
        p = Problem(kind, V, 9, top, 2.0, alpha, skip=0.0)
        j = np.arange(top)
        p.ids[0] = 17
        p.ids[1] = j // 2 % V
        p.ids[2] = j % 7
        p.ids[3] = (j * 256) % V
        p.ids[4] = np.where(j % 3 == 0, V - 1, j % V)
        p.ids[5] = np.where(j % 2 == 0, -1, V)
        p.ids[6] = np.where(j < top - 2, j % V, p.ids[6, 0])
        p.labels[:7] = [17, 3, 20, 256 % V, V - 1, 5, V // 2]
        a = p.run()
        check(p, a)
        b = p.run(in_place=True)
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


@pytest.mark.parametrize("V", [500, 50000])
def test_repeated_and_missing_entries(hip, V):
    """One token several times in a row, ids outside of the vocabulary, rows without any entry."""
    announce(f"distill entries V={V}")
    for alpha in (1.0, 0.4):
        p = Problem("f32", V, 30, 9, 2.0, alpha, skip=0.1)
        p.ids[0] = p.ids[0, 0]
        p.ids[1, 3:] = p.ids[1, 0]
        p.ids[2, 4] = -1
        p.ids[3, 5:] = V
        p.ids[4] = -7
        p.ids[5] = np.iinfo(np.int32).max
        p.ids[6, 1:] = np.iinfo(np.int32).min
        p.labels[:8] = 3
        p.ids[0, 2] = p.labels[0]
        check(p)
        p.ids[:] = -1
        check(p)


@pytest.mark.parametrize("V", [100, 40000])
def test_no_row_counted(hip, V):
    announce(f"distill nothing counted V={V}")
    p = Problem("bf16", V, 11, 5)
    p.labels[:] = -1
    loss, d = p.run()
    assert np.array_equal(loss, np.zeros(4, np.float32)) and not d.any()


@pytest.mark.parametrize("V", [600, 60000])
def test_masked_vocabulary_and_uncounted_rows(hip, V):
    """-inf logits are tokens that cannot occur, far finite ones nearly so; rows not counted may hold anything."""
    announce(f"distill masked V={V}")
    rng = np.random.default_rng(8)
    for low in (-np.inf, -1e9, float(np.finfo(np.float32).min)):
        for tau, alpha in ((2.0, 0.5), (3.0, 0.5), (1.0, 1.0)):
            p = Problem("f32", V, 13, 8, tau, alpha, skip=0.4)
            out = rng.random((p.T, V)) < 0.7
            out[:, :8] = False
            for t in range(p.T):
                out[t, p.ids[t]] = False
            out[np.arange(p.T), np.maximum(p.labels, 0)] = False
            p.logits = np.where(out, low, p.logits).astype(np.float32)
            p.l64 = p.logits.astype(np.float64)
            wl, wd = p.want()
            p.logits[p.labels < 0] = np.nan
            loss, d = p.run()
            tol = (60 + 16 * np.sqrt(V)) * U32 * 4
            assert np.allclose(loss, wl, rtol=tol, atol=tol), (low, tau, loss, wl)
            assert np.all(np.isfinite(d)) and not d[p.labels < 0].any()
            assert np.allclose(d, wd, rtol=0, atol=tol)
            assert not d[out].any()


@pytest.mark.parametrize("V", [600, 60000])
def test_rows_far_from_zero(hip, V):
    """Logits around +-1e4 and +-1e30 keep their differences: exact in float, as the row's largest is taken off first."""
    announce(f"distill far V={V}")
    for off, step in ((1e4, 2.0 ** -8), (-1e4, 2.0 ** -8), (1e30, 0.0), (-1e30, 0.0)):
        for tau, alpha in ((2.0, 0.5), (1.0, 0.5), (3.0, 0.9)):
            p = Problem("f32", V, 6, 5, tau, alpha)
            p.logits = (np.round(p.logits / max(step, 1)) * step + off).astype(np.float32)
            p.l64 = p.logits.astype(np.float64)
            check(p)


@pytest.mark.parametrize("V", [600, 60000])
def test_values_that_are_not_finite(hip, V):
    """As a log-softmax has it: an infinite or NaN logit, a row of -inf, a label past the vocabulary make the loss
    NaN; a teacher's token that the student finds impossible makes it infinite, one that the teacher does takes no part."""
    announce(f"distill not finite V={V}")
    for change in ("inf", "nan", "all", "label", "teacher"):
        p = Problem("f32", V, 9, 6, skip=0.0)
        if change == "inf":
            p.logits[5, 7] = np.inf
        elif change == "nan":
            p.logits[5, V - 1] = np.nan
        elif change == "all":
            p.logits[5] = -np.inf
        elif change == "label":
            p.labels[5] = V
        else:
            p.teacher[5, 2] = np.nan
        loss, d = p.run()
        assert np.isnan(loss[0]), change
        ok = np.ones(9, bool)
        ok[5] = False
        assert np.all(np.isfinite(d[ok])), change
    p = Problem("f32", V, 9, 6, skip=0.0)
    p.logits[4, p.ids[4, 1]] = -np.inf
    p.labels[4] = (p.ids[4, 1] + 1) % V
    p.l64 = p.logits.astype(np.float64)
    loss, d = p.run()
    assert loss[0] == np.inf and loss[1] == np.inf and np.isfinite(loss[2]) and np.all(np.isfinite(d))
    p.teacher[4, 1] = -np.inf
    p.z64 = p.teacher.astype(np.float64)
    loss, d = p.run()
    wl, wd = p.want()
    assert np.all(np.isfinite(loss)) and np.allclose(loss, wl, rtol=1e-4) and np.allclose(d, wd, atol=1e-5)


def test_label_past_the_vocabulary_counts_by_its_sign_alone(hip):
    announce("distill alpha 1 labels")
    p = Problem("f32", 300, 9, 6, 2.0, 1.0, skip=0.3)
    p.labels[p.labels >= 0] = 5000
    check(p)


def test_gradient_against_differences(hip):
    """The loss of logits moved either way along a direction. A second difference over the step bounds what the first
    leaves out; float losses add their rounding."""
    announce("distill differences")
    rng = np.random.default_rng(12)
    for tau, alpha in ((2.0, 0.5), (1.0, 1.0), (3.0, 0.8)):
        p = Problem("f32", 50, 25, 6, tau, alpha)
        p.dloss[:] = 1
        d = p.run()[1].astype(np.float64)
        base = p.logits.copy()
        for _ in range(3):
            step = rng.standard_normal(base.shape).astype(np.float32)
            eps = 2.0 ** -5
            at = []
            for k in (eps, -eps, 2 * eps, -2 * eps):
                p.logits = base + np.float32(k) * step
                at.append(float(p.run()[0][0]))
            first, wide = (at[0] - at[1]) / (2 * eps), (at[2] - at[3]) / (4 * eps)
            assert abs(first - (d * step).sum()) <= abs(first - wide) + 64 * U32 * max(map(abs, at)) / eps
        p.logits = base


@pytest.mark.parametrize("V,T", [(700, 2100), (70000, 6)])
def test_same_bits_every_time_and_captured(hip, V, T):
    announce(f"distill same bits V={V}")
    rt = runtime()
    p = Problem("bf16", V, T, 16)
    first = p.run()
    s = Stream()
    again = [p.run(), p.run(stream=s.handle)]
    assert all(np.array_equal(a, b) for other in again for a, b in zip(first, other))
    fwd, back, loss, d, stats, keep = p.views()
    graph, exe = C.c_void_p(), C.c_void_p()
    assert rt.hipStreamBeginCapture(C.c_void_p(s.handle), 0) == 0
    try:
        H.distill_loss(*fwd, s.handle)
        H.distill_loss_back(*back, s.handle)
    finally:
        rc = rt.hipStreamEndCapture(C.c_void_p(s.handle), C.byref(graph))
    assert rc == 0 and rt.hipGraphInstantiate(C.byref(exe), graph, None, None, 0) == 0
    for _ in range(3):
        H.fill_f32(loss.ptr, 0.0, 4)
        p.run()
        assert rt.hipGraphLaunch(exe, C.c_void_p(s.handle)) == 0
        H.sync(s.handle)
        assert np.array_equal(loss.read(), first[0]) and np.array_equal(d.read(), first[1])
    rt.hipGraphExecDestroy(exe)
    rt.hipGraphDestroy(graph)
    for k in keep:
        k.free()
    s.close()
