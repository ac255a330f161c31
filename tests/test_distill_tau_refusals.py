"""Temperatures that the distillation loss cannot compute with: the kernels' factor on a logit is log2 e / tau in 32 bits, and where
that is infinite every term would be NaN. Refused before any device work."""
import numpy as np
import pytest

from test_fp8_distill_refusals import loss, loss_args, loss_back, refused
from traincpp_amd import hip as H


@pytest.mark.parametrize("tau", [3.0e-39, 3.5e-39, 4.2e-39])
def test_temperatures_whose_factor_is_infinite(tau):
    with np.errstate(over="ignore"):
        assert np.isfinite(np.float32(1) / np.float32(tau)) and np.isinf(np.float32(1.44269504) / np.float32(tau))
    for call in (loss, loss_back):
        refused(call, {**loss_args(), "tau": tau}, H.E_INVALID)
