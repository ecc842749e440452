"""Sampling at temperatures at which one step of a logit is many powers of two
of mass, up to where the largest value has all of it; uncut rows, whose masses
are summed without bins, among them.

Tolerances as in test_gpu_sample: u lies in the middle of an interval of at
least 2^-21 of the kept mass, masses are off by 2^-33 of themselves and half a
unit of 2^-36 of twice the largest, logprob by half a step of fp32 and 2^-21."""
import numpy as np
import pytest

import test_gpu_sample as G

pytestmark = pytest.mark.gpu

COLD = [1e-5, 1e-6, 1e-7, 3e-8, 1e-8, 3e-9, 2e-9, 1e-9, 1e-10, 1e-11]
# maxima at which the lowest counted value lies at different places
TOPS = [5.0, 8.0, 10.0, 12.5, 15.0, 30.0, -3.0]


def _rows(rng, N, dtype, device, scale=1.0):
    """Ordinary logits, rows with columns masked out or not a number, each under
    a largest value that one to three columns hold, and a near neighbour."""
    import torch
    v = np.minimum(rng.standard_normal((len(TOPS), N)) * 2, 4.0)
    for m, top in enumerate(TOPS):
        v[m] = np.minimum(v[m], top - 1)
        at = rng.choice(N, 4, replace=False)
        v[m, at[:1 + m % 3]] = top
        v[m, at[3]] = np.nextafter(np.float32(top), np.float32(-np.inf))
    v = v * scale
    v[1, rng.random(N) < 0.9] = -np.inf
    v[1, N - 1] = TOPS[1] * scale
    v[2, 1000:3000] = -np.inf
    return torch.from_numpy(v.astype(np.float32)).to(dtype).to(device)


def _one(logits, T, which, times, seed):
    """The rows `times` over (more rows: another launch plan)."""
    import torch
    rng = np.random.default_rng(seed)
    rows = G._np(logits)
    T = float(np.float32(T))
    ks = [{'k': 5, 'kp': 3}.get(which, 0)] * len(rows)
    ps = [0.9 if 'p' in which else 1.0] * len(rows)
    qs = [0.01 if 'q' in which else 0.0] * len(rows)
    us, cols = zip(*[G._place(rng, row, T, k, float(np.float32(p)), float(np.float32(q)))
                     for row, k, p, q in zip(rows, ks, ps, qs)])
    n = len(rows) * times
    # (uncut calls: no setting but the temperature)
    cut = [x * times for x in (ks, ps, qs)] if which else [None] * 3
    token, logprob, flags = G._run(logits.repeat(times, 1), list(us) * times, [T] * n, *cut, workspace_fill=0xff)
    for m, row in enumerate(rows):
        tok, lp = G.S.sample(row, T, ks[m], float(np.float32(ps[m])), float(np.float32(qs[m])), float(us[m]))
        assert tok == cols[m] and (token[m::len(rows)] == tok).all(), (T, m, token[m::len(rows)], tok)
        off = np.abs(logprob[m::len(rows)] - lp)
        assert (off <= 2.0 ** -24 * abs(lp) + 2.0 ** -21).all(), (T, m, off, lp)
    assert flags == 0


@pytest.mark.parametrize('dtype', ['bf16', 'fp32'])
@pytest.mark.parametrize('N', [8192, 8193, 20003, 50001])
@pytest.mark.parametrize('times', [1, 10])
@pytest.mark.parametrize('which', ['', 'k', 'p', 'q'])
def test_small_temperatures(device, dtype, N, times, which):
    """7 and 70 rows: up to 256 parts in a call, and more."""
    logits = _rows(np.random.default_rng(N), N, G._dtype(dtype), device)
    for T in COLD:
        print(f'{dtype} N={N} times={times} {which} T={T}', flush=True)
        _one(logits, T, which, times, N + times)


@pytest.mark.parametrize('scale', [1e6, 1e8, 1e9, 1e10, 1e12])
@pytest.mark.parametrize('which', ['', 'p'])
def test_large_logits(device, scale, which):
    logits = _rows(np.random.default_rng(3), 20003, G._dtype('fp32'), device, scale)
    for times in (1, 15):
        _one(logits, 1.0, which, times, 5)


@pytest.mark.parametrize('T', [1e-38, 1e-40, 1e-43])
def test_smallest_temperatures_on_small_logits(device, T):
    """Subnormal temperatures, logits some of them large."""
    logits = _rows(np.random.default_rng(4), 20003, G._dtype('fp32'), device, T * 4)
    for times in (1, 15):
        for which in ('', 'k'):
            _one(logits, T, which, times, 6)


def test_masked_columns_at_a_small_temperature(device):
    """-inf and NaN columns and a short last part add nothing to an uncut row."""
    import torch
    rng = np.random.default_rng(7)
    N = 8192 * 3 + 5
    logits = _rows(rng, N, G._dtype('fp32'), device)
    logits[3, 17::2] = float('nan')
    logits[4, :8192] = -float('inf')
    logits[5, 8192:] = -float('inf')
    logits[:, 3] = logits.nan_to_num(-float('inf')).amax(1)
    rows = G._np(logits)
    for T in (1e-8, 2e-9):
        us = [G._place(rng, np.where(np.isnan(row), -np.inf, row), float(np.float32(T)), 0, 1.0, 0.0)[0] for row in rows]
        for times in (1, 10):
            token, logprob, flags = G._run(logits.repeat(times, 1), us * times, [T] * (7 * times))
            assert flags == 1
            for i in range(7 * times):
                row = np.where(np.isnan(rows[i % 7]), -np.inf, rows[i % 7])
                tok, lp = G.S.sample(row, float(np.float32(T)), u=float(us[i % 7]))
                assert token[i] == tok and abs(logprob[i] - lp) <= 2.0 ** -24 * abs(lp) + 2.0 ** -21, (T, i)
