"""The preference loss over logits (trc_hip_preference_loss) and its gradient against
64 bits.

Tolerance: lse is a float near its value: one rounding of it, one of the logarithm, and the
relative error of a sum of V positive terms, each an exponential of a rounded difference:
(|lse| + log V + 4 + |l| spread) 2^-24 covers them with the sum's 8 sqrt(n) of n terms a thread
(see test_gpu_lora.py). logp adds one lse error per counted token. A gradient is off by the relative
error of exp(l - lse), that of lse and of the rounded difference, and of the weight; 16 bits round it
once more."""
import numpy as np
import pytest

from conftest import announce
from gpu_util import Dev, Stream
from traincpp_amd import hip as H
from tuning_util import TYPES, U32, Mat, decode, encode, starts, vec

pytestmark = pytest.mark.gpu

HALF = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


class Problem:
    def __init__(self, kind, V, lens, seed=3, prompt=0.25, beta=0.1, smoothing=0.0, pad=0, lead=0):
        rng = np.random.default_rng(seed)
        self.kind, self.V, self.lens, self.beta, self.smoothing = kind, V, list(lens), beta, smoothing
        self.T, self.P, self.pad, self.lead = max(int(sum(lens)), 1), len(lens) // 2, pad, lead
        self.logits, self.l64 = encode(rng.standard_normal((self.T, V)) * 3, kind)
        self.labels = rng.integers(0, V, self.T).astype(np.int32)
        self.start = starts(lens)
        for lo, n in zip(self.start, self.lens):
            self.labels[lo:lo + int(n * prompt)] = -1
        self.ref = (-np.log(V) * np.array(self.lens) + rng.standard_normal(len(lens)) * 3).astype(np.float32)
        self.dloss = np.array([0.7], np.float32)

    def run(self, stream=None, in_place=False, twice=False):
        t = TYPES[self.kind]
        keep = []

        def v(x, kind=H.TYPE_F32):
            d, out = vec(x, kind)
            keep.append(d)
            return d, out

        m = Mat(self.logits, t, self.pad, self.lead)
        d = m if in_place else Mat(np.zeros_like(self.logits), t, self.pad, self.lead)
        keep += [m, d]
        _, labels = v(self.labels, H.TYPE_I32)
        _, start = v(self.start.astype(np.int32), H.TYPE_I32)
        _, ref = v(self.ref)
        _, dloss = v(self.dloss)
        nan = lambda n: v(np.full(n, np.nan, np.float32))
        lse, logp, slope, loss = nan(self.T), nan(2 * self.P), nan(self.P), nan(1)
        H.preference_loss(m.t, labels, start, ref, self.beta, self.smoothing, lse[1], logp[1], slope[1], loss[1], stream)
        H.preference_loss_back(m.t, labels, start, lse[1], slope[1], dloss, self.beta, d.t, stream)
        H.sync(stream)
        out = [k.read() for k in (lse[0], logp[0], slope[0], loss[0])] + [d.read()]
        for k in keep:
            k.free()
        return out

    def want(self):
        with np.errstate(all="ignore"):
            top = self.l64.max(1, keepdims=True)
            lse = (top + np.log(np.exp(self.l64 - top).sum(1, keepdims=True)))[:, 0]
            counted = self.labels >= 0
            logp = np.zeros(2 * self.P)
            seq = np.full(self.T, -1)
            for s in range(2 * self.P):
                for t in range(self.start[s], self.start[s + 1]):
                    seq[t] = s
                    if counted[t]:
                        logp[s] += self.l64[t, self.labels[t]] - lse[t] if self.labels[t] < self.V else np.nan
            gap = logp - self.ref
            z = self.beta * (gap[0::2] - gap[1::2])
            up, down = np.logaddexp(0, -z), np.logaddexp(0, z)
            e = self.smoothing
            loss = np.mean((1 - e) * up + (e * down if e else 0))
            sig = lambda q: np.where(q >= 0, 1 / (1 + np.exp(-np.abs(q))), np.exp(-np.abs(q)) / (1 + np.exp(-np.abs(q))))
            slope = e * sig(z) - (1 - e) * sig(-z)
            d = np.zeros_like(self.l64)
            for t in range(self.T):
                if seq[t] < 0 or not counted[t]:
                    continue
                w = float(self.dloss[0]) * self.beta / self.P * slope[seq[t] // 2] * (-1 if seq[t] % 2 else 1)
                d[t] = -w * np.exp(self.l64[t] - lse[t])
                if self.labels[t] < self.V:
                    d[t, self.labels[t]] += w
            return np.where(counted, lse, 0.0), logp, slope, loss, d, seq


def check(p, **kw):
    lse, logp, slope, loss, d = p.run(**kw)
    wlse, wlogp, wslope, wloss, wd, seq = p.want()
    spread = np.abs(p.l64).max()
    e_lse = (np.abs(wlse).max() + np.log(p.V) + 4 + spread + 8 * np.sqrt(p.V)) * U32
    assert np.abs(lse - wlse).max() <= e_lse
    counts = np.array([(p.labels[a:b] >= 0).sum() for a, b in zip(p.start, p.start[1:])])
    e_logp = counts * e_lse
    assert np.all(np.abs(logp - wlogp) <= e_logp + 2 * U32 * np.abs(wlogp)), "logp"
    e_z = p.beta * (e_logp[0::2] + e_logp[1::2]) + U32
    assert np.all(np.abs(slope - wslope) <= e_z / 4 + 4 * U32), "slope"
    assert abs(loss[0] - wloss) <= e_z.max() + 4 * U32 * abs(wloss), "loss"
    got = decode(d, p.kind)
    unit = float(np.abs(p.dloss[0])) * p.beta / p.P
    e_w = unit * (e_z.max() / 4 + 8 * U32)
    prob = np.where((wd != 0) | (seq >= 0)[:, None], np.exp(p.l64 - np.where(p.labels >= 0, wlse, np.inf)[:, None]), 0)
    bound = (prob + (p.labels[:, None] == np.arange(p.V))) * (e_w + unit * (e_lse + (spread * 4 + 8) * U32)) \
        + HALF[p.kind] * np.abs(wd) + (2.0 ** -25 if p.kind == "f16" else 1e-36)
    over = np.abs(got - wd) / bound
    assert over.max() <= 1, f"dlogits: {over.max()} of the bound at {np.unravel_index(over.argmax(), over.shape)}"
    out = (p.labels < 0) | (seq < 0)
    assert not got[out].any()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("V,lens", [
    (1, [2, 3]), (2, [1, 1]), (7, [4, 5, 1, 2]), (1000, [9, 12, 30, 1]), (4099, [3, 6]), (32000, [17, 8]),
    (50001, [5, 4, 3, 2]), (131071, [2, 3]), (333, [200, 150, 1, 97, 64, 64]),
])
def test_loss_and_gradient(hip, kind, V, lens):
    announce(f"preference {kind} V={V} {lens}")
    check(Problem(kind, V, lens, smoothing=0.1 if V % 2 else 0.0))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("pad,lead", [(1, 1), (3, 5), (8, 8)])
def test_strided_rows(hip, kind, pad, lead):
    announce(f"preference strides {kind} {pad} {lead}")
    check(Problem(kind, 8209, [4, 7], pad=pad, lead=lead))
    check(Problem(kind, 515, [4, 7], pad=pad, lead=lead), in_place=True)


@pytest.mark.parametrize("lens", [[0, 3], [3, 0], [0, 0], [0, 0, 5, 2], [40, 0, 0, 1]])
def test_empty_sequences(hip, lens):
    announce(f"preference empty {lens}")
    check(Problem("f32", 100, lens))


def test_no_token_counted(hip):
    announce("preference nothing counted")
    p = Problem("bf16", 300, [5, 6])
    p.labels[:] = -1
    check(p)
    p = Problem("bf16", 40000, [5, 6])
    p.labels[:] = -100
    check(p)


@pytest.mark.parametrize("beta,gap", [(0.1, 0), (1.0, 400), (1.0, -400), (5.0, 3000), (0.0, 10)])
@pytest.mark.parametrize("smoothing", [0.0, 0.3, 1.0])
def test_far_apart_pairs(hip, beta, gap, smoothing):
    """Large ratios either way: the loss grows linearly and the slope keeps its bits."""
    announce(f"preference far apart {beta} {gap} {smoothing}")
    p = Problem("f32", 64, [4, 5], beta=beta, smoothing=smoothing)
    p.ref[0] -= gap
    check(p)


def test_rows_in_no_sequence(hip):
    announce("preference rows outside")
    p = Problem("f32", 90, [6, 7])
    p.start = np.array([2, 6, 11], np.int32)
    check(p)


@pytest.mark.parametrize("V", [600, 60000])
def test_masked_vocabulary_and_uncounted_rows(hip, V):
    """-inf logits are tokens that cannot occur; rows not counted may hold anything."""
    announce(f"preference masked V={V}")
    p = Problem("f32", V, [6, 7], prompt=0.5)
    rng = np.random.default_rng(8)
    p.l64 = p.l64.copy()
    out = rng.random((p.T, V)) < 0.7
    out[np.arange(p.T), np.maximum(p.labels, 0)] = False
    p.logits = np.where(out, -np.inf, p.logits).astype(np.float32)
    p.logits[3] = np.where(np.arange(V) == p.labels[3], p.logits[3], np.finfo(np.float32).min)
    p.l64 = p.logits.astype(np.float64)
    want = p.want()
    p.logits[p.labels < 0] = np.nan
    lse, logp, slope, loss, d = p.run()
    assert np.allclose(lse, want[0], rtol=0, atol=(40 + 8 * np.sqrt(V)) * U32)
    assert np.allclose(logp, want[1], rtol=0, atol=10 * (40 + 8 * np.sqrt(V)) * U32)
    assert np.all(np.isfinite(d)) and not d[p.labels < 0].any()
    assert np.allclose(d, want[4], rtol=0, atol=(60 + 8 * np.sqrt(V)) * U32)
    assert not d[out & (p.labels >= 0)[:, None]].any()


@pytest.mark.parametrize("V", [600, 60000])
def test_values_that_are_not_finite(hip, V):
    """As a log-softmax has it: an infinite or NaN logit, a row of -inf and a label past the
    vocabulary make the loss NaN; a label whose logit is -inf makes its sequence's logp -inf."""
    announce(f"preference not finite V={V}")
    for change in ("inf", "nan", "all", "label"):
        p = Problem("f32", V, [6, 7])
        if change == "inf":
            p.logits[5, 7] = np.inf
        elif change == "nan":
            p.logits[5, V - 1] = np.nan
        elif change == "all":
            p.logits[5] = -np.inf
        else:
            p.labels[5] = V
        lse, logp, slope, loss, d = p.run()
        assert np.isnan(loss[0]) and np.isnan(slope[0]) and np.isnan(logp[0]) and np.isfinite(logp[1]), change
    for at, sign in ((5, np.inf), (12, -np.inf)):  # the chosen answer cannot occur; the rejected one cannot
        p = Problem("f32", V, [6, 7])
        p.logits[at, p.labels[at]] = -np.inf
        p.l64 = p.logits.astype(np.float64)
        lse, logp, slope, loss, d = p.run()
        assert logp[0 if at == 5 else 1] == -np.inf
        assert loss[0] == (np.inf if sign > 0 else 0.0) and slope[0] == (-1.0 if sign > 0 else 0.0)
        assert np.all(np.isfinite(d))


def test_gradient_against_differences(hip):
    """The loss of logits moved either way along a direction. A second difference of the loss
    over the step bounds what the first leaves out; float losses add their rounding."""
    announce("preference differences")
    rng = np.random.default_rng(12)
    p = Problem("f32", 50, [7, 9, 5, 4], beta=0.5, smoothing=0.1)
    p.dloss[:] = 1
    d = p.run()[4].astype(np.float64)
    base = p.logits.copy()
    for _ in range(4):
        step = rng.standard_normal(base.shape).astype(np.float32)
        eps = 2.0 ** -6
        at = []
        for k in (eps, -eps, 2 * eps, -2 * eps):
            p.logits = base + np.float32(k) * step
            at.append(float(p.run()[3][0]))
        first, wide = (at[0] - at[1]) / (2 * eps), (at[2] - at[3]) / (4 * eps)
        # (an error of order eps^2 grows fourfold when the step doubles)
        assert abs(first - (d * step).sum()) <= abs(first - wide) + 64 * U32 * max(map(abs, at)) / eps


def test_sums_of_long_sequences(hip):
    """Sequences whose sums are thousands of times the ratios between them."""
    announce("preference long sequences")
    p = Problem("f32", 260, [6000, 5500], beta=0.1)
    want = p.want()
    p.ref[:] = want[1].astype(np.float32) + np.array([1.5, -0.5], np.float32)
    check(p)


def test_same_bits_every_time(hip):
    announce("preference same bits")
    for V in (700, 70000):
        p = Problem("bf16", V, [11, 9])
        first = p.run()
        s = Stream()
        again = [p.run(), p.run(stream=s.handle)]
        s.close()
        for other in again:
            assert all(np.array_equal(a, b) for a, b in zip(first, other))
