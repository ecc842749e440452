"""Adapters whose values leave the finite range somewhere, against the definition
in 64 bits: a result is infinite, NaN or finite where base + scale * sum_r B v is,
whatever the 16-bit numbers are that v is cut into.

Whole numbers and powers of two make every finite result exact: |v| <= 2 K = 128,
sums below 2^24.  The definition is summed term by term, so that 0 times inf is a
NaN of its own column and row alone."""
import numpy as np
import pytest

import test_gpu_adapter as A

pytestmark = pytest.mark.gpu

INF = float('inf')


def _definition(c):
    x, a, b, base, scales = (c[n].double().cpu().numpy() for n in ('x', 'a', 'b', 'base', 'scales'))
    ids, R, out = c['ids'].cpu().numpy(), c['rank'], base.copy()
    with np.errstate(invalid='ignore', over='ignore'):
        for i in np.unique(ids[ids >= 0]):
            at, n0 = np.flatnonzero(ids == i), 0
            v = np.stack([(x[at] * row).sum(1) for row in a[i]], 1)
            for p, width in enumerate(c['slices']):
                for n in range(n0, n0 + width):
                    out[at, n] += scales[i] * (b[i, n] * v[:, p * R:(p + 1) * R]).sum(1)
                n0 += width
    return out


def _check(c, got):
    import torch
    out, flags = got
    with np.errstate(over='ignore'):
        want = torch.from_numpy(_definition(c)).to(out.dtype).double().numpy()
    got = out.double().cpu().numpy()
    wrong = ~((got == want) | (np.isnan(got) & np.isnan(want)))
    assert not wrong.any(), (np.argwhere(wrong)[:5], got[wrong][:5], want[wrong][:5])
    touched = want[c['ids'].cpu().numpy() >= 0]
    assert flags == (0 if np.isfinite(touched).all() else 4 if out.dtype == torch.float32 else 12)
    return got


# rows, columns, inputs, rank, slots, slices
SHAPES = [(1, 100, 64, 16, 1, 1), (9, 77, 64, 8, 2, 2), (40, 130, 64, 24, 3, 1), (64, 64, 64, 64, 4, 1), (100, 90, 64, 40, 2, 2),
          (300, 200, 64, 16, 3, 1), (33, 90, 64, 128, 3, 1), (90, 70, 64, 72, 2, 2), (500, 65, 64, 200, 2, 1),
          (4100, 70, 64, 64, 3, 1), (1100, 70, 64, 128, 3, 1)]
TYPES = [('bf16', 'bf16'), ('bf16', 'fp32'), ('fp16', 'fp16'), ('fp16', 'fp32')]


@pytest.mark.parametrize('dtype,out_type', TYPES)
@pytest.mark.parametrize('M,N,K,R,slots,parts', SHAPES)
def test_infinities_in_b(device, dtype, out_type, M, N, K, R, slots, parts):
    """inf times a v that its first 16-bit number holds, and times one that it does not."""
    import torch
    print(f'adapter inf {dtype} {out_type} M={M} N={N} R={R}', flush=True)
    rng = np.random.default_rng(M + N + R)
    c = A._case(rng, M, N, K, R, slots, parts, dtype, out_type, device, True, ldb=N + 3)
    c['x'][::3] *= 0.5
    # (v = 257 and 2049 + 1/2 and the like: beyond one number of 8 and of 11 bits, either side of it)
    c['a'][:, ::2, 0] = 2049.0 if dtype == 'fp16' else 514.0
    c['x'][:, 0] = torch.where(c['x'][:, 0] == 0, 1, c['x'][:, 0])
    c['b'][:, ::5] = torch.where(c['b'][:, ::5] > 0, 1, 0).to(c['b'].dtype)
    plain, flags = A._run(c)
    assert flags in (0, 8)
    hit = torch.from_numpy(np.sort(rng.choice(N, max(1, N // 7), replace=False))).to(device)
    for n in hit.tolist():
        r = int(rng.integers(R))
        c['b'][:, n, r] = INF if n % 2 else -INF
        if n % 3 == 0:
            c['b'][:, n, (r + 1) % R] = INF
    for in_place in (False, True):
        got = A._run(c, in_place)
        _check(c, got)
        rest = torch.ones(N, dtype=torch.bool, device=device)
        rest[hit] = False
        assert torch.equal(got[0][:, rest], plain[:, rest])        # no other column sees it


@pytest.mark.parametrize('dtype,out_type', TYPES)
@pytest.mark.parametrize('M,R', [(5, 16), (80, 64), (300, 24), (20, 128), (1100, 72)])
def test_an_infinite_v_beside_others(device, dtype, out_type, M, R):
    """inf in A: v of one r infinite, the others as they are, up to past fp16's range."""
    import torch
    rng = np.random.default_rng(M + R)
    c = A._case(rng, M, 90, 64, R, 2, 1, dtype, out_type, device, True)
    c['a'][:, 3, 5] = INF
    c['x'][:, 5] = torch.where(c['x'][:, 5] == 0, 1, c['x'][:, 5])
    c['x'][0] = 1
    c['a'][:, 4] = 2048.0                              # v up to 2^17
    c['b'][:, :, 3] = torch.where(c['b'][:, :, 3] == 0, 1, c['b'][:, :, 3])
    c['b'][:, ::3, 3] = 0                              # 0 times inf
    got = _check(c, A._run(c))
    ids = c['ids'].cpu().numpy()
    assert np.isinf(got[ids >= 0][:, 1::3]).all() and np.isnan(got[ids >= 0][:, ::3]).all()


@pytest.mark.parametrize('M,R', [(5, 16), (80, 64), (300, 24), (20, 128), (1100, 72)])
def test_infinities_times_a_v_far_below_the_largest(device, M, R):
    """fp16 rows whose v lie 2^50 apart: the smaller is not 0."""
    import torch
    c = A._case(np.random.default_rng(M), M, 70, 64, R, 2, 1, 'fp16', 'fp32', device, True, ids=np.arange(M) % 2)
    c['x'].fill_(1)
    c['a'].zero_()
    c['b'].zero_()
    c['scales'].fill_(1)
    c['a'][:, 0, :] = 32768.0                          # v = 2^21
    c['a'][:, 1, 7] = 2.0 ** -24
    c['a'][:, 2, 7] = -2.0 ** -24
    c['b'][:, ::4, 1] = INF
    c['b'][:, 1::4, 2] = INF
    c['b'][:, 2::4, 3] = INF                           # v = 0: NaN
    c['b'][:, 3::4, 0] = 2.0
    got = _check(c, A._run(c))
    assert (got[:, ::4] == INF).all() and (got[:, 1::4] == -INF).all() and np.isnan(got[:, 2::4]).all()
    assert np.isfinite(got[:, 3::4]).all()


@pytest.mark.parametrize('out_type', ['bf16', 'fp32'])
@pytest.mark.parametrize('M,R', [(5, 16), (80, 64), (300, 24), (20, 128), (1100, 72)])
def test_finite_results_of_a_v_near_the_end_of_the_range(device, out_type, M, R):
    """v between bf16's largest value and fp32's, and scale v past both: the results are finite."""
    import torch
    c = A._case(np.random.default_rng(M), M, 70, 64, R, 2, 1, 'bf16', out_type, device, True, ids=np.arange(M) % 2)
    c['x'].zero_()
    c['x'][:, 0], c['x'][:, 1] = 2.0 ** 100, 2.0 ** 91
    c['a'].zero_()
    c['b'].zero_()
    c['base'].zero_()
    c['a'][:, 1, 0] = c['a'][:, 1, 1] = 255 * 2.0 ** 20            # v = 255 (2^120 + 2^111): rounds to 2^128
    c['a'][:, 2, 0] = 2.0 ** 20
    c['b'][0, :, 1] = 2.0 ** -60
    c['b'][1, :, 2] = 2.0 ** -60
    c['scales'].copy_(torch.tensor([1.0, 2.0 ** 10]))
    got = _check(c, A._run(c))
    assert np.isfinite(got).all() and (got[1::2] == 2.0 ** 70).all()


@pytest.mark.parametrize('M,R', [(40, 16), (300, 64), (40, 128)])
def test_other_rows_keep_their_results(device, M, R):
    """Rows of a tile that hold infinities and NaN leave the others bit for bit."""
    import torch
    c = A._case(np.random.default_rng(7), M, 130, 264, R, 2, 2, 'bf16', 'fp32', device, False, ids=np.arange(M) % 2)
    want, flags = A._run(c)
    assert flags == 0
    c['x'][3, 9] = INF
    c['x'][8] = float('nan')
    c['x'][17, 200] = -INF
    got, flags = A._run(c)
    assert flags == 4
    rest = [m for m in range(M) if m not in (3, 8, 17)]
    assert torch.equal(got[rest], want[rest])
    assert not bool(got[[3, 8, 17]].isfinite().any())
