"""Greedy rows take the first maximum whatever their other settings hold (a
request of temperature 0 often comes with a top_p of 0)."""
import numpy as np
import pytest

import test_gpu_sample as G

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('N,times', [(300, 1), (8192, 1), (9000, 1), (40000, 8)])
def test_settings_of_greedy_rows_do_not_matter(device, N, times):
    rng = np.random.default_rng(N)
    odd = [(0.0, 0.0, 0.5), (1.0, 0.0, 1.0), (1.0, -1.0, 0.5), (np.nan, 0.0, 0.5), (1.0, np.nan, np.nan), (2.0, 3.0, -4.0),
           (0.9, 0.1, np.inf)]
    logits = G._logits(rng, len(odd), N, G._dtype('bf16'), device)
    best = G._np(logits).argmax(1)
    p, q, u = zip(*odd)
    for T in (0.0, -0.0):
        n = len(odd) * times
        token, logprob, flags = G._run(logits.repeat(times, 1), u * times, [T] * n, [3] * n, p * times, q * times)
        assert (token == np.tile(best, times)).all() and (logprob == 0).all() and flags == 0
