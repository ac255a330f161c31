"""Rows of the distillation gradient (trc_hip_distill_loss_back) that test_gpu_distill.py's comparisons leave open."""
import numpy as np
import pytest

from conftest import announce
from test_gpu_distill import HALF, Problem
from tuning_util import TYPES, U32, decode, encode

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("V", [3, 500, 50000])
@pytest.mark.parametrize("in_place", [False, True])
def test_label_past_the_vocabulary(hip, V, kind, in_place):
    """It makes the loss NaN, and its row's gradient too; the other rows' gradients are those beside an ordinary label. With
    alpha = 1 it counts by its sign alone."""
    announce(f"distill label past the vocabulary V={V} {kind} in_place={in_place}")
    for alpha, tau in ((0.4, 2.0), (0.0, 1.0), (0.7, 3.0), (0.5, 1.0), (1.0, 2.0)):
        p = Problem(kind, V, 9, 3, tau, alpha, skip=0.0)
        p.labels[5] = V - 1
        loss, d = p.run(in_place=in_place)
        for label in (V, np.iinfo(np.int32).max):
            p.labels[5] = label
            got_loss, got = p.run(in_place=in_place)
            ok = np.arange(9) != 5
            assert np.array_equal(got[ok], d[ok])
            if alpha == 1:
                assert np.array_equal(got_loss, loss) and np.array_equal(got, d)
            else:
                assert np.isnan(got_loss[0]) and np.isnan(got_loss[2]) and got_loss[3] == 9
                assert np.isnan(decode(got[5], kind)).all(), (alpha, tau, label)


@pytest.mark.parametrize("V", [600, 60000])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_masked_vocabulary_token_by_token(hip, V, kind):
    """Logits of tokens that cannot occur (-inf, or nearly so), whole rows and rows in parts: every element of the gradient within its
    own bound, test_gpu_distill.py's with the spread of what is not masked; masked tokens have none."""
    announce(f"distill masked, token by token V={V} {kind}")
    rng = np.random.default_rng(18)
    for low in (-np.inf, -1e9, -3e38):
        for tau, alpha in ((2.0, 0.5), (3.0, 0.5), (1.0, 1.0)):
            p = Problem(kind, V, 13, 8, tau, alpha, skip=0.4)
            out = rng.random((p.T, V)) < 0.7
            out[:, :8] = False
            for t in range(p.T):
                out[t, p.ids[t]] = False
            out[np.arange(p.T), np.maximum(p.labels, 0)] = False
            out[3, V // 3:] = True  # a row whose later parts have nothing left
            out[3, p.ids[3]] = False
            out[3, max(p.labels[3], 0)] = False
            out[4, p.ids[4, 2]] = True  # the teacher finds it impossible as well
            if p.labels[4] == p.ids[4, 2]:
                p.labels[4] = p.ids[4, 3]
            p.teacher, p.z64 = p.teacher.copy(), p.z64.copy()
            p.teacher[4, 2] = p.z64[4, 2] = -np.inf
            p.logits, p.l64 = encode(np.where(out, np.float32(low), p.l64), kind)
            wl, wd = p.want()
            nan = np.array([np.nan], np.float32) if kind == "f32" else np.array([0x7FC0], np.uint16)
            p.logits[p.labels < 0] = nan[0]
            loss, d = p.run()
            got, n = decode(d, kind), wl[3]
            e_s = 2 * (np.ptp(p.l64[~out]) / min(tau, 1) + 8 * np.sqrt(V) + 8) * U32
            zs = np.ptp(p.z64[np.isfinite(p.z64)])
            assert loss[3] == n
            for i in (1, 2):
                assert abs(loss[i] - wl[i]) <= e_s + 2 * U32 * abs(wl[i])
            mag = np.zeros_like(wd)
            for t in np.nonzero(p.labels >= 0)[0]:
                for x, w in ((p.l64[t] / tau, alpha * tau), (p.l64[t], 1 - alpha)):
                    mag[t] += w * np.exp(x - x.max()) / np.exp(x - x.max()).sum()
                z = np.exp((p.z64[t] - p.z64[t].max()) / tau)
                np.add.at(mag[t], p.ids[t], alpha * tau * z / z.sum())
                mag[t, p.labels[t]] += 1 - alpha
            err = mag * (abs(float(p.dloss[0])) / n) * (2 * e_s + (zs / tau + 16 + p.top) * U32)
            bound = err + HALF[kind] * (np.abs(wd) + err) + 1e-36
            over = np.abs(got - wd) / bound
            assert over.max() <= 1, (low, tau, over.max(), np.unravel_index(over.argmax(), over.shape))
            assert not got[p.labels < 0].any() and not got[out].any()
