"""Probabilities where softcap / temperature is below f32's range."""
import numpy as np
import pytest

import kv8_ref as ref
from test_gpu_sample import run_probs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cap,temperature", [(1e-37, 1e10), (1e-30, 1e16), (1e-37, 3e38), (2e-38, 1e7), (1.0, 3e38), (0.0, 3e38)])
@pytest.mark.parametrize("vocab", [997, 4096, 5001])
def test_probabilities_of_vanishing_units(gpu, cap, temperature, vocab):
    # the soft-capped logits differ by nothing: what is not masked is even, what is masked is 0
    rng = np.random.default_rng(vocab)
    x = (rng.standard_normal((4, vocab)) * 4).astype(np.float32)
    x[1, rng.random(vocab) < 0.5] = -np.inf
    x[2] = -np.inf
    x[3, 7] = np.nan
    want, bound = ref.probabilities(x[:3], cap, temperature)
    got = run_probs(gpu, x, cap, temperature)
    assert np.isnan(got[3]).all()
    assert np.all(np.abs(got[:3] - want) <= bound * want)
    assert not got[2].any() and not got[1][np.isinf(x[1])].any()
