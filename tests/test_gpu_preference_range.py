"""The preference loss's sums over logits of every size that a finite float has: rows most of
which a finite value masks, and rows whose first tokens lie far from the others.

Tolerance, per row: terms more than 100 below the row's largest are less than 1e-43 of it and do not
count. Of the others each is an exponential whose argument is at most 100 in magnitude and rounded three
times at most (the difference, its product, what a join adds), so off by 300 * 2^-24; the sum of V
positive terms and its float have the (|lse| + log V + 4 + 8 sqrt(V)) 2^-24 of
test_gpu_preference.py. The gradient's exponentials have the same arguments."""
import numpy as np
import pytest

from conftest import announce
from gpu_util import Dev
from traincpp_amd import hip as H
from tuning_util import TYPES, U32, Mat, decode, encode, vec

pytestmark = pytest.mark.gpu

HALF = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
BETA, SMOOTHING, DLOSS = 0.2, 0.1, 0.7


def check(kind, logits, labels, T, far=False, in_place=False):
    """`logits` are the counted rows, a sequence each; the batch has T rows, of which the others are in no
    sequence (they decide in how many parts a row is summed). far: lse's own rounding to a float, |lse| 2^-24,
    counts in full in lse alone, elsewhere as of 1024 at most."""
    n, V = logits.shape
    assert n % 2 == 0 and T >= n
    held, l = encode(logits, kind)
    whole = np.zeros((T, V), held.dtype)
    whole[:n] = held
    y = np.full(T, -1, np.int32)
    y[:n] = labels
    with np.errstate(under="ignore"):
        top = l.max(1)
        log_s = np.log(np.exp(l - top[:, None]).sum(1))
        prob = np.exp((l - top[:, None]) - log_s[:, None])
    lse = top + log_s
    logp = (l[np.arange(n), labels] - top) - log_s
    rng = np.random.default_rng(1)
    ref = (logp + rng.standard_normal(n)).astype(np.float32)
    z = BETA * ((logp - ref)[0::2] - (logp - ref)[1::2])
    slope = SMOOTHING / (1 + np.exp(-z)) - (1 - SMOOTHING) / (1 + np.exp(z))
    loss = np.mean((1 - SMOOTHING) * np.logaddexp(0, -z) + SMOOTHING * np.logaddexp(0, z))
    unit = DLOSS * BETA / (n // 2)
    w = unit * np.stack([slope, -slope], 1).reshape(-1, 1)
    at = labels[:, None] == np.arange(V)
    d = w * (at - prob)

    t, keep = TYPES[kind], []

    def v(x, type_=H.TYPE_F32):
        dev, out = vec(x, type_)
        keep.append(dev)
        return dev, out

    m = Mat(whole, t)
    dl = m if in_place else Mat(np.zeros_like(whole), t)
    keep += [m, dl]
    _, yt = v(y, H.TYPE_I32)
    _, start = v(np.arange(n + 1, dtype=np.int32), H.TYPE_I32)
    _, rt = v(ref)
    _, dt = v(np.array([DLOSS], np.float32))
    out = [v(np.full(k, np.nan, np.float32)) for k in (T, n, n // 2, 1)]
    H.preference_loss(m.t, yt, start, rt, BETA, SMOOTHING, *(o[1] for o in out))
    H.preference_loss_back(m.t, yt, start, out[0][1], out[2][1], dt, BETA, dl.t)
    H.sync()
    glse, glogp, gslope, gloss = (o[0].read() for o in out)
    gd = dl.read()
    for k in keep:
        k.free()

    sums = (300 + np.log(V) + 4 + 8 * np.sqrt(V)) * U32
    e_lse = sums + np.abs(lse) * U32

    def near(got, want, bound, what):
        with np.errstate(invalid="ignore"):
            over = np.abs(got.astype(np.float64) - want) / bound
        bad = ~(over <= 1)
        assert not bad.any(), f"{what}: {got[bad][:4]} for {want[bad][:4]} at {np.argwhere(bad)[:4].tolist()}"

    near(glse[:n], lse, e_lse, "lse")
    if far:
        e_lse = sums + np.minimum(np.abs(lse), 1024) * U32
    assert not glse[n:].any()
    e_logp = e_lse + 2 * U32 * np.abs(logp)
    near(glogp, logp, e_logp, "logp")
    e_z = BETA * (e_logp[0::2] + e_logp[1::2]) + U32
    near(gslope, slope, e_z / 4 + 4 * U32, "slope")
    near(gloss, np.array([loss]), e_z.max() + 4 * U32 * abs(loss), "loss")
    bound = (prob + at) * unit * (np.repeat(e_z, 2)[:, None] / 4 + 8 * U32 + e_lse[:, None] + 400 * U32) \
        + HALF[kind] * np.abs(d) + (2.0 ** -25 if kind == "f16" else 1e-36)
    near(decode(gd[:n], kind), d, bound, "dlogits")
    assert not gd[n:].any()


# (V, T) by type: a row in one part, and in several; in each a thread has its first loads and more
ONE = {"f32": (8191, 40), "f16": (17000, 2048), "bf16": (17000, 2048)}
PARTS = {"f32": (60000, 40), "f16": (60001, 512), "bf16": (60001, 512)}


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("sizes", [ONE, PARTS], ids=["one", "parts"])
def test_finite_masks(hip, kind, sizes):
    """A finite value far below stands for a token that cannot occur, and covers all that a thread reads:
    all but the last 40 tokens, or runs of a few thousand."""
    V, T = sizes[kind]
    announce(f"preference finite masks {kind} V={V} T={T}")
    rng = np.random.default_rng(4)
    masks = [-7e3, -1e6, -1e9, -3e10, -1e11, -1e12, -7e12, -1e15, -1e20, -1e25, -3e30, -1e38, -1.7e38, -2.2e38]
    for runs in (False, True):
        l = rng.standard_normal((len(masks), V)) * 2
        out = np.arange(V) < V - 40 if not runs else (np.arange(V) // 3000) % 2 == 0
        out[V - 1] = False
        labels = np.where(rng.random(len(masks)) < 0.5, V - 1, np.flatnonzero(~out)[0]).astype(np.int32)
        check(kind, np.where(out, np.array(masks)[:, None], l), labels, T)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_rows_masked_but_for_their_label(hip, kind):
    announce(f"preference rows of one token {kind}")
    for V, T in (ONE[kind], PARTS[kind]):
        masks = np.array([-1e4, -1e8, -1e10, -1e11, -1e12, -1e13, -1e16, -1e38])
        l = np.repeat(masks[:, None], V, 1)
        labels = np.array([0, V - 1, 5, V // 2, V - 3, 17, 4096, 1], np.int32)
        l[np.arange(len(masks)), labels] = np.linspace(-4, 4, len(masks))
        check(kind, l, labels, T)


FAR = [60, 70] + list(range(76, 91)) + [100]
FIRST = {"f32": 4096, "f16": 8192, "bf16": 8192}  # what a workgroup's first loads hold


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("sizes", [ONE, PARTS], ids=["one", "parts"])
@pytest.mark.parametrize("part", ["first", "half", "spread"])
def test_first_tokens_far_below(hip, kind, sizes, part):
    """A run of tokens at the row's start (what the first loads hold, or every second thread's share of it,
    or such a run in every part), 60 to 100 below the others."""
    V, T = sizes[kind]
    announce(f"preference first tokens below {kind} V={V} T={T} {part}")
    rng = np.random.default_rng(6)
    l = rng.standard_normal((len(FAR), V))
    i, lane = np.arange(V), 4 if kind == "f32" else 8
    out = i < FIRST[kind] if part != "spread" else i % (FIRST[kind] * 3 // 2) < FIRST[kind]
    if part == "half":
        out &= (i // lane) % 2 == 0
    l -= out * np.array(FAR, np.float64)[:, None]
    labels = np.where(rng.random(len(FAR)) < 0.7, V - 1, 3).astype(np.int32)
    check(kind, l, labels, T)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("sizes", [ONE, PARTS], ids=["one", "parts"])
def test_few_late_tokens_far_above(hip, kind, sizes):
    """Rows of zeros with a few tokens, behind what the first loads hold, 40 to 89 above."""
    V, T = sizes[kind]
    announce(f"preference late tokens above {kind} V={V} T={T}")
    rng = np.random.default_rng(7)
    tops = [40, 60, 80, 84, 86, 87, 87.5, 88, 88.3, 88.6, 88.7, 89]
    l = np.zeros((len(tops) * 2, V))
    for r in range(len(l)):
        at = FIRST[kind] + rng.choice(V - FIRST[kind], 8 if r % 2 else 64, replace=False)
        l[r, at] = tops[r // 2]
    labels = l.argmax(1).astype(np.int32)
    labels[::5] = 0
    check(kind, l, labels, T)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("sizes", [ONE, PARTS, {k: (1000, 40) for k in TYPES}], ids=["one", "parts", "short"])
def test_rows_far_from_zero(hip, kind, sizes, in_place):
    """A row's log-sum may be so large that its float holds little of the sum, or nothing: rows all of whose
    tokens a finite value masks, and rows moved as a whole. Their probabilities are those of the
    differences between their logits."""
    V, T = sizes[kind]
    announce(f"preference far from zero {kind} V={V} T={T} in place {in_place}")
    rng = np.random.default_rng(9)
    at = np.array([2e3, -5e3, 3e4, -6e4] + ([] if kind == "f16" else [1e5, -1e6, -1e9, 3e12, -1e20, -1e30, 2e38, -3e38]))
    even = np.repeat(at[:, None], V, 1)  # every token alike
    moved = even + rng.standard_normal(even.shape) * 2
    spread = even * (1 + (rng.random(even.shape) < 0.3) * 2.0 ** -6)
    near_bound = 1024 + np.array([-60.0, -12, -11, -10, 2, 50])[:, None] + rng.standard_normal((6, V))
    l = np.concatenate([even, moved, spread, near_bound])
    labels = np.where(rng.random(len(l)) < 0.5, l.argmax(1), rng.integers(0, V, len(l))).astype(np.int32)
    # (where the label lies far under the row's largest, the loss is that distance: not what is looked at here)
    low = l[np.arange(len(l)), labels] < l.max(1) - 50
    labels[low] = l.argmax(1)[low]
    check(kind, l, labels, max(T, 64), far=True, in_place=in_place)
