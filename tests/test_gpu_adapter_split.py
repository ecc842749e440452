"""Every 16-bit number that v is cut into reaches the result, beside its own r.

v is a whole number of 24 bits, v = 2^16 a + 2^8 b + c with |a| in 128..255, formed
exactly (three products, their sums below 2^24); each column of B has one entry, 1 or
-1, so a result is base + scale * v[r] of one r.  fp32 results: three parts of bf16
hold v, two of fp16 hold it to 2^-23; the sum of three products loses at most 2^-23 of
itself at each of its additions (the matrix cores may cut), and the base's addition
half a step.  In all 5 * 2^-23 of |scale v| and 2^-24 of the result.  Fewer
parts miss by up to 2^-17 (two of bf16) and 2^-12 (one of fp16): the test says how
many of its results would be off by more than is allowed.

bf16 results of two parts: the base is -(scale v) rounded, so the result is what the
first part leaves, to 2^-17 of |v| and half a step of itself."""
import numpy as np
import pytest

import test_gpu_adapter as A

pytestmark = pytest.mark.gpu

# rows, columns, inputs, rank, slots, slices: ranks of 1 to 12 pieces of 8, in one launch and in two
SHAPES = [(1, 70, 24, 8, 1, 1), (5, 130, 24, 16, 3, 1), (40, 90, 256, 24, 2, 2), (64, 64, 24, 32, 4, 1), (100, 150, 24, 40, 3, 1),
          (200, 300, 24, 64, 2, 3), (300, 90, 24, 16, 5, 1), (1121, 130, 24, 24, 3, 2), (500, 140, 24, 56, 3, 1), (4100, 70, 24, 40, 3, 1),
          (4099, 130, 24, 64, 2, 1), (7, 200, 24, 72, 3, 1), (90, 130, 24, 96, 2, 2), (300, 200, 24, 200, 3, 1), (1100, 130, 24, 128, 3, 1),
          (1500, 100, 24, 72, 3, 2)]


def _dtype(name):
    return A._dtype(name)


def _case(rng, M, N, K, R, slots, parts, dtype, out_type, device):
    """(case, scale v of each result in float64)."""
    import torch
    groups = 8
    abc = rng.integers(128, 256, (M, groups, 3)) * rng.choice((-1, 1), (M, groups, 3))
    xs = np.zeros((M, K))
    xs[:, :24] = (abc * np.array([256, 256, 1])).reshape(M, 24)
    v = (abc * np.array([65536, 256, 1])).sum(2)                       # of each group of three inputs
    a = np.zeros((slots, parts * R, K))
    of = rng.integers(0, groups, (slots, parts * R))                   # the group that a row of A takes
    s, r = np.meshgrid(np.arange(slots), np.arange(parts * R), indexing='ij')
    for j, by in enumerate((256, 1, 1)):
        a[s, r, 3 * of + j] = by
    ends = np.sort(rng.integers(0, N + 1, parts - 1)).tolist() + [N]
    slices = tuple(int(w) for w in np.diff([0] + ends))
    part = np.searchsorted(ends, np.arange(N), side='right')
    at = np.stack([rng.permutation(np.arange(N) % R) for _ in range(slots)])       # the r of each column
    sign = rng.choice((-1, 1), (slots, N))
    b = np.zeros((slots, N, R))
    b[np.arange(slots)[:, None], np.arange(N)[None], at] = sign
    scales = 2.0 ** rng.integers(-3, 3, slots)
    ids = rng.integers(0, slots, M)
    row = part[None] * R + at                                          # of A, for each slot and column
    want = scales[ids][:, None] * sign[ids] * v[np.arange(M)[:, None], of[ids[:, None], row[ids]]]

    def tensor(t, kind):
        return torch.from_numpy(t.astype(np.float32)).to(_dtype(kind)).to(device)
    base = np.round(rng.standard_normal((M, N)) * 1000) if out_type == 'fp32' else -want
    c = dict(x=tensor(xs, dtype), a=tensor(a, dtype), b=tensor(b, dtype), scales=tensor(scales, 'fp32'),
             ids=torch.from_numpy(ids.astype(np.int32)).to(device), base=tensor(base, out_type), slices=slices, rank=R,
             dtype=dtype, out_type=out_type)
    return c, want


def _parts(v, dtype, count):
    """v as the sum of `count` 16-bit numbers (fp16: within its range already)."""
    import torch
    left, total = torch.from_numpy(v), torch.zeros(v.shape, dtype=torch.float64)
    for _ in range(count):
        p = left.to(_dtype(dtype)).double()
        total, left = total + p, left - p
    return total.numpy()


@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
@pytest.mark.parametrize('M,N,K,R,slots,parts', SHAPES)
def test_fp32_results(device, dtype, M, N, K, R, slots, parts):
    print(f'split {dtype} M={M} N={N} R={R}', flush=True)
    c, sv = _case(np.random.default_rng(M + N + R), M, N, K, R, slots, parts, dtype, 'fp32', device)
    base = c['base'].double().cpu().numpy()
    tol = 5 * 2.0 ** -23 * np.abs(sv) + 2.0 ** -24 * np.abs(base + sv)
    # Would one part fewer be seen?  Two of bf16 are off by up to 64 units of 2^-23 of v's binade where the first
    # leaves more than half of what it can (half of all v), 32 for a quarter of them, ..; twice the tolerance is 10 to
    # 20 such units, so about half of many results are seen, and some of a few.
    fewer = _parts(sv * 2.0 ** -13, dtype, 2 if dtype == 'bf16' else 1) * 2.0 ** 13
    assert (np.abs(fewer - sv) > 2 * tol).mean() > 0.1
    for in_place in (False, True):
        out, flags = A._run(c, in_place)
        got = out.double().cpu().numpy()
        bad = np.abs(got - (base + sv)) > tol
        assert flags == 0 and not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], (base + sv)[bad][:5])


@pytest.mark.parametrize('M,N,K,R,slots,parts', SHAPES)
def test_bf16_results(device, M, N, K, R, slots, parts):
    c, sv = _case(np.random.default_rng(M + N + R), M, N, K, R, slots, parts, 'bf16', 'bf16', device)
    want = c['base'].double().cpu().numpy() + sv
    tol = 2.0 ** -17 * np.abs(sv) + 5 * 2.0 ** -23 * np.abs(sv) + 2.0 ** -9 * np.abs(want)
    assert (np.abs(want) > 2 * tol).mean() > 0.5                       # (one part leaves 0)
    out, flags = A._run(c)
    bad = np.abs(out.double().cpu().numpy() - want) > tol
    assert flags == 0 and not bad.any(), (np.argwhere(bad)[:5], out.double().cpu().numpy()[bad][:5], want[bad][:5])
