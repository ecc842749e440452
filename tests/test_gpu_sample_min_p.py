"""min-p where the largest logit and T ln q nearly cancel: the least value that
is kept lies next to 0, where fp32's steps are far smaller than what is known of
mx + T ln q.

Kept and dropped values are at least 1e-6 from the border: a relative 1e-6 / T
in mass, against 2^-52 |mx| / T of rounding.  u and logprob as in
test_gpu_sample."""
import numpy as np
import pytest

import test_gpu_sample as G

pytestmark = pytest.mark.gpu

# largest value, T, q: none of the 64 values around the estimate is kept, or all are
CASES = [(3.390625, 1.3, 0.0736690015), (3.8533942699432373, 0.9850131869316101, 0.02),
         (2.870436668395996, 1.2466148138046265, 0.1), (2.4376869201660156, 0.7342647910118103, 0.03615638613700867),
         (0.5917440056800842, 0.5305120348930359, 0.3277774155139923),
         (1.1432390213012695, 1.465924859046936, 0.45846304297447205),
         (0.6115639805793762, 0.3085101842880249, 0.13775014877319336),
         (1.318121314048767, 1.3338487148284912, 0.3722427785396576),
         (0.8883882164955139, 0.8603029251098633, 0.3560636341571808)]


def _rows(rng, N, cases):
    rows = np.empty((len(cases), N), np.float32)
    for m, (top, _, _) in enumerate(cases):
        rows[m] = rng.choice([top * 0.75, top / 4, 1e-3, 1e-6, -1e-6, -1e-3, -top / 4, -2 * top], N,
                             p=[.05, .05, .1, .1, .1, .1, .2, .3])
        rows[m, rng.integers(N)] = top
    return rows


@pytest.mark.parametrize('N,times', [(40, 1), (8192, 1), (9000, 1), (40001, 8)])
@pytest.mark.parametrize('which', ['q', 'kq', 'pq'])
def test_border_next_to_zero(device, N, times, which):
    import torch
    rng = np.random.default_rng(N + len(which))
    logits = torch.from_numpy(_rows(rng, N, CASES)).to(device)
    rows = G._np(logits)
    T, q = [float(np.float32(c[1])) for c in CASES], [float(np.float32(c[2])) for c in CASES]
    k = [3 + N // 10 if 'k' in which else 0] * len(CASES)
    p = [0.999 if 'p' in which else 1.0] * len(CASES)
    us = []
    for m, row in enumerate(rows):
        # the last kept of the lowest value: what a border at the top would have dropped
        cols, e = G.S.kept(row, T[m], k[m], float(np.float32(p[m])), q[m])
        col = int(cols[e == e.min()][-1])
        assert len(cols) > 1 and (row[cols] > 0).all() and e.min() >= 2 * G.MARGIN * e.sum()
        us.append(np.float32(G.S.uniform_for(row, T[m], k[m], float(np.float32(p[m])), q[m], col)[0]))
    G._check(logits.repeat(times, 1), T * times, k * times, p * times, q * times, us * times)


def test_border_next_to_zero_of_16_bit_rows(device):
    """A bf16 maximum, few live columns: the case of a shortlist."""
    import torch
    logits = torch.full((2, 12), -5.0, dtype=torch.bfloat16, device=device)
    logits[:, 4] = 3.390625
    logits[:, [2, 7, 9]] = 1.0
    T, q = [1.2999999523162842] * 2, [0.0736690015] * 2
    rows = G._np(logits)
    us = [np.float32(G.S.uniform_for(row, T[0], 0, 1.0, float(np.float32(q[0])), col)[0]) for row, col in zip(rows, (2, 9))]
    G._check(logits, T, [0] * 2, [1.0] * 2, q, us, [2, 9])


@pytest.mark.parametrize('dtype', ['bf16', 'fp16', 'fp32'])
def test_borders_anywhere(device, dtype):
    """Largest values and q of every size: the border far from its estimate's
    scale, below the lowest value, at the largest."""
    import torch
    rng = np.random.default_rng(12)
    M, N = 60, 700
    base = rng.standard_normal((M, N)) * 10.0 ** rng.uniform(-3, 3, (M, 1))
    base[::4] = np.abs(base[::4])
    base[1::4] = -np.abs(base[1::4])
    base[2::8] = np.round(base[2::8])
    logits = torch.from_numpy(base.astype(np.float32)).to(G._dtype(dtype)).to(device)
    rows = G._np(logits)
    Ts, qs, us, cols = [], [], [], []
    for m, row in enumerate(rows):
        T = float(np.float32(10.0 ** rng.uniform(-2, 2)))
        e = np.unique(G.S.masses(row, G.S.order(row), T))
        e = e[e >= 1e-12]
        i = int(rng.integers(len(e)))
        # in the middle between two masses; 1, and far below all
        q = [float(np.float32((e[i] + (e[i - 1] if i else 0)) / 2)), 1.0, 1e-20][m % 7 // 5 + (m % 7 == 6)]
        if len(e) > 1 and q < 1 and np.abs(e - q).min() <= 2.0 ** -20 * q:
            q = 1e-20
        u, col = G._place(rng, row, T, 0, 1.0, q)
        for l, v in zip((Ts, qs, us, cols), (T, q, u, col)):
            l.append(v)
    G._check(logits, Ts, [0] * M, [1.0] * M, qs, us, cols)
