"""Adapters of many requests against their definition in 64 bits.

Whole numbers (x and A in -1..1 and -2..2, B in -2..2, power-of-two scales) make
every product and sum exact: |v| <= 2 K < 2^16 (the two halves of v hold 16
bits), sums below 2^24.  Those compare bit for bit with the rounded 64-bit result.

Ordinary values: v's sums of K terms |x A| lose at most 2^-23 each (the matrix
cores may truncate), K + 8 additions (of which the error bound takes the sum of
all |x A|); its two halves 2^-17 (bf16) or 2^-22 (fp16) of the largest |v| of the
row and slice; the second product's 2 R additions 2^-23 of the sum of |B v|; scale,
base: 2^-23 of the result's terms.  Then half a step of the output's type."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF_STEP = {'bf16': 2.0 ** -8, 'fp16': 2.0 ** -11, 'fp32': 2.0 ** -24}
HALVES = {'bf16': 2.0 ** -17, 'fp16': 2.0 ** -22}


def _dtype(name):
    import torch
    return {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}[name]


def _case(rng, M, N, K, R, slots, parts, dtype, out_type, device, exact, ids=None, ldx=0, ldb=0):
    import torch
    t = _dtype(dtype)
    if parts == 1:
        slices = (N,)
    else:
        cuts = np.sort(rng.integers(0, N + 1, parts - 1))
        slices = tuple(int(v) for v in np.diff(np.concatenate([[0], cuts, [N]])))
    if exact:
        xs, A, B = rng.integers(-1, 2, (M, K)), rng.integers(-2, 3, (slots, parts * R, K)), rng.integers(-2, 3, (slots, N, R))
        scales, base = 2.0 ** rng.integers(-2, 1, slots), rng.integers(-50, 51, (M, N))
    else:
        xs, A = rng.standard_normal((M, K)), rng.standard_normal((slots, parts * R, K)) / np.sqrt(max(K, 1))
        B, scales, base = rng.standard_normal((slots, N, R)), rng.uniform(0.25, 2.0, slots), rng.standard_normal((M, N))
    if ids is None:
        ids = rng.integers(-1, slots, M) if slots else np.full(M, -1)
    x = torch.full((M, ldx or K), 7.0, dtype=t, device=device)
    x[:, :K] = torch.from_numpy(xs.astype(np.float32))
    wide = torch.full((M, ldb or N), 3.0, dtype=_dtype(out_type), device=device)
    wide[:, :N] = torch.from_numpy(base.astype(np.float32))
    return dict(x=x[:, :K], a=torch.from_numpy(A.astype(np.float32)).to(t).to(device),
                b=torch.from_numpy(B.astype(np.float32)).to(t).to(device),
                scales=torch.from_numpy(scales.astype(np.float32)).to(device),
                ids=torch.from_numpy(np.asarray(ids).astype(np.int32)).to(device), base=wide[:, :N], slices=slices,
                rank=R, dtype=dtype, out_type=out_type)


def _run(c, in_place=False, ldo=0):
    import torch
    from ornith_g256 import native
    M, N = c['base'].shape
    dev = c['x'].device
    buf = torch.full((M, max(ldo, N)), -7.0, dtype=c['base'].dtype, device=dev)
    out = buf[:, :N]
    if in_place:
        out.copy_(c['base'])
    flags = torch.zeros(1, dtype=torch.int32, device=dev)
    ws = torch.full((native.adapter_bytes(M, c['a'].shape[1]),), 0xff, dtype=torch.uint8, device=dev)
    native.adapter_out(c['x'], c['a'], c['b'], c['scales'], c['ids'], None if in_place else c['base'], out, ws, flags,
                       slices=c['slices'])
    torch.cuda.synchronize()
    assert bool((buf[:, N:] == -7.0).all())
    return out, int(flags)


def _want(c):
    """(result, bound on the error before the last rounding) in float64."""
    x, a, b, base = (c[n].double().cpu().numpy() for n in ('x', 'a', 'b', 'base'))
    scales, ids, R = c['scales'].double().cpu().numpy(), c['ids'].cpu().numpy(), c['rank']
    K = x.shape[1]
    out, err = base.copy(), np.zeros_like(base)
    for i in np.unique(ids):
        if i < 0 or i >= len(scales):
            continue
        at = ids == i
        v = x[at] @ a[i].T
        dv = (K + 8) * 2.0 ** -23 * (np.abs(x[at]) @ np.abs(a[i]).T)
        n0 = 0
        for p, width in enumerate(c['slices']):
            cols, of = slice(n0, n0 + width), slice(p * R, (p + 1) * R)
            vp, bp = v[:, of], b[i, cols]
            d = dv[:, of] + HALVES[c['dtype']] * (np.abs(vp).max(1, keepdims=True) + dv[:, of])
            delta, mass = vp @ bp.T, (np.abs(vp) + d) @ np.abs(bp).T
            out[at, cols] += scales[i] * delta
            err[at, cols] = scales[i] * (d @ np.abs(bp).T + (2 * R + 1) * 2.0 ** -23 * mass)
            n0 += width
    err += 2.0 ** -23 * (np.abs(out) + err) * (ids >= 0)[:, None]
    return out, err


def _check(c, got, flags=0, exact=False):
    import torch
    out, seen = got
    assert seen == flags
    want, err = _want(c)
    none = c['ids'].cpu().numpy() < 0
    assert torch.equal(out[torch.from_numpy(none)].cpu(), c['base'][torch.from_numpy(none)].cpu())
    got = out.double().cpu().numpy()
    if exact:
        assert np.abs(want).max(initial=0) < 2 ** 22
        rounded = torch.from_numpy(want).to(out.dtype).double().numpy()
        assert (got == rounded).all(), (np.argwhere(got != rounded)[:5], got[got != rounded][:5], rounded[got != rounded][:5])
        return
    tol = err + HALF_STEP[c['out_type']] * (np.abs(want) + err)
    if c['out_type'] == 'fp16':
        tol = tol + 2.0 ** -25
    bad = np.abs(got - want) > tol
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], tol[bad][:5])
    # the bound is loose by the square root of its length: the mean error is far below it
    ref = np.sqrt((want ** 2).mean()) if want.size else 0
    if want.size > 64:
        assert np.sqrt(((got - want) ** 2).mean()) <= ref * (HALF_STEP[c['out_type']] + 2.0 ** -17)


# rows, columns, inputs, rank, slots, slices
SHAPES = [(1, 1, 8, 8, 1, 1), (1, 100, 64, 8, 3, 1), (1, 6144, 2048, 16, 4, 1), (2, 15, 40, 16, 2, 2), (3, 64, 520, 24, 5, 1),
          (5, 257, 136, 40, 2, 3), (16, 128, 256, 16, 1, 1), (17, 130, 264, 8, 1, 2), (32, 1000, 512, 64, 16, 1),
          (40, 77, 2120, 32, 40, 8), (64, 1024, 2048, 64, 16, 2), (65, 513, 1000, 16, 7, 1), (77, 5003, 136, 24, 6, 1),
          (130, 200, 4096, 8, 3, 3), (256, 320, 1024, 16, 200, 1), (300, 2048, 512, 128, 4, 1), (1121, 192, 264, 16, 3, 1),
          (2100, 100, 64, 8, 2, 2), (5000, 70, 72, 16, 17, 1), (9, 300, 32768, 8, 2, 1), (33, 90, 128, 512, 3, 1),
          (7, 40, 64, 256, 2, 3), (4, 70000, 64, 8, 2, 1),
          # tiles of 32 rows, and of 64 above rank 64
          (4100, 90, 136, 64, 3, 2), (4099, 200, 72, 40, 5, 1), (4200, 64, 1096, 56, 2, 1), (1100, 130, 264, 128, 3, 1),
          (1500, 70, 72, 72, 5, 2), (2000, 300, 64, 120, 40, 1)]


@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
@pytest.mark.parametrize('M,N,K,R,slots,parts', SHAPES)
def test_whole_numbers(device, dtype, M, N, K, R, slots, parts):
    print(f'adapter {dtype} M={M} N={N} K={K} R={R} slots={slots} parts={parts}', flush=True)
    rng = np.random.default_rng(M * 31 + N * 7 + K + R)
    ldx, ldb, ldo = K + 8 * (N % 3), N + M % 5, N + (N + M) % 4
    # |B v| sums stay below 2^22: a third of x and of B is zero, so v is near sqrt(K) and sums near sqrt(R K) * 2
    c = _case(rng, M, N, K, R, slots, parts, dtype, 'fp32', device, True, ldx=ldx, ldb=ldb)
    _check(c, _run(c, ldo=ldo), exact=True)
    _check(c, _run(c, in_place=True, ldo=ldo), exact=True)
    c = _case(rng, M, N, K, R, slots, parts, dtype, dtype, device, True)
    _check(c, _run(c), exact=True)
    _check(c, _run(c, in_place=True), exact=True)


@pytest.mark.parametrize('dtype,out_type', [('bf16', 'bf16'), ('bf16', 'fp32'), ('fp16', 'fp16'), ('fp16', 'fp32'), ('bf16', 'fp16'),
                                            ('fp16', 'bf16')])
@pytest.mark.parametrize('M,N,K,R,slots,parts', SHAPES)
def test_rows(device, dtype, out_type, M, N, K, R, slots, parts):
    rng = np.random.default_rng(M + N + K + R)
    c = _case(rng, M, N, K, R, slots, parts, dtype, out_type, device, False, ldb=N + M % 3)
    _check(c, _run(c, in_place=bool(M % 2)))


@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
@pytest.mark.parametrize('pattern', ['one', 'none', 'runs', 'each', 'one row', 'alternating', 'first and last'])
@pytest.mark.parametrize('M', [1, 16, 31, 64, 65, 200, 1500])
def test_id_patterns(device, dtype, pattern, M):
    rng = np.random.default_rng(M)
    slots = 70
    ids = {'one': np.full(M, 3), 'none': np.full(M, -1), 'runs': np.sort(rng.integers(-1, 5, M))[::-1],
           'each': np.arange(M) % slots, 'one row': np.where(np.arange(M) == M // 2, 69, -1),
           'alternating': np.where(np.arange(M) % 2, 0, 69), 'first and last': np.where(np.arange(M) % (M - 1 or 1), -5, 7)}[pattern]
    c = _case(rng, M, 136, 128, 16, slots, 1, dtype, 'fp32', device, True, ids=ids)
    _check(c, _run(c), exact=True)
    _check(c, _run(c, in_place=True), exact=True)


@pytest.mark.parametrize('M', [5, 100])
def test_ids_past_the_slots(device, M):
    import torch
    rng = np.random.default_rng(2)
    ids = rng.integers(-1, 3, M)
    ids[3] = 3
    ids[4] = 2 ** 31 - 1
    c = _case(rng, M, 100, 64, 8, 3, 1, 'bf16', 'bf16', device, True, ids=ids)
    for in_place in (False, True):
        out, flags = _run(c, in_place)
        assert flags == 16
        assert torch.equal(out[3:5], c['base'][3:5])
        _check(c | dict(ids=torch.where(c['ids'] > 2, -1, c['ids'])), (out, 0), exact=True)


@pytest.mark.parametrize('M', [6, 90])
def test_a_row_does_not_depend_on_the_others(device, M):
    import torch
    rng = np.random.default_rng(3)
    c = _case(rng, M, 200, 264, 16, 3, 2, 'bf16', 'fp32', device, False)
    c['ids'][:6] = torch.tensor([1, 1, 0, 1, -1, 2])
    full, flags = _run(c)
    assert flags == 0
    c['x'][1] = float('nan')
    c['x'][3] = float('inf')
    c['x'][4] = float('nan')                           # has no adapter
    some, flags = _run(c)
    assert flags == 4
    rest = [m for m in range(M) if m not in (1, 3)]
    assert torch.equal(some[rest], full[rest])
    assert bool(some[1].isnan().all()) and not bool(some[3].isfinite().any())


def test_large_and_small_values(device):
    """v past fp16's range, and far below it; a non-finite 16-bit result."""
    import torch
    rng = np.random.default_rng(4)
    for M in (3, 80):
        for by in (2.0 ** 12, 2.0 ** -18):
            c = _case(rng, M, 90, 1024, 16, 2, 1, 'fp16', 'fp32', device, False)
            c['x'].mul_(by)
            c['a'].mul_(32)
            c['scales'].mul_(1 / by / 32)
            # (fp16's subnormal x are not changed again: the definition takes them as they are)
            _check(c, _run(c))
        c = _case(rng, M, 90, 1024, 16, 2, 1, 'fp16', 'fp16', device, False, ids=np.zeros(M))
        c['b'].mul_(2.0 ** -16)                        # subnormal B
        c['scales'].mul_(2.0 ** 16)
        _check(c, _run(c))
        c['scales'].fill_(1e9)
        out, flags = _run(c)
        assert flags == 8 and not bool(out.isnan().any()) and bool(out.isinf().any())


def test_empty_calls(device):
    import torch
    rng = np.random.default_rng(5)
    for M, N, K, slots in ((0, 40, 64, 2), (3, 0, 64, 2), (3, 40, 0, 2), (3, 40, 64, 0), (90, 40, 0, 2), (90, 40, 64, 0)):
        c = _case(rng, M, N, K, 8, slots, 1, 'bf16', 'bf16', device, True)
        for in_place in (False, True):
            out, flags = _run(c, in_place)
            assert flags == 0 and torch.equal(out, c['base'])
