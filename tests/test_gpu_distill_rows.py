"""Rows of the distillation gradient (trc_hip_distill_loss_back) that test_gpu_distill.py's comparisons leave open."""
import numpy as np
import pytest

from conftest import announce
from test_gpu_distill import Problem
from tuning_util import TYPES, decode

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
