"""Plain 4-bit linears against their definition in 64 bits.

Whole-number rows (-3..3) with power-of-two scales make every product and sum
exact in fp32 (below 2^24 units), so those compare bit for bit with the rounded
64-bit result.  Ordinary rows: each fp32 operation is off by at most 2^-23 of
its result (the matrix cores may truncate), a term passes at most 128 additions
in its group's block, a multiply-add each for z, s and every 128-k block, and 8
to join the waves; what is added is at most 32 |s x| a term.  Then half a step
of the output's type."""
import numpy as np
import pytest

from oracle import w4 as O

pytestmark = pytest.mark.gpu

HALF_STEP = {'bf16': 2.0 ** -8, 'fp16': 2.0 ** -11, 'fp32': 2.0 ** -24}


def _dtype(name):
    import torch
    return {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}[name]


def _case(rng, M, N, K, group, zeros, dtype, device, exact, ldx=0):
    import torch
    words = rng.integers(0, 2 ** 32, (N, K // 8), dtype=np.uint32)
    groups = -(-K // group)
    if exact:
        x = rng.integers(-3, 4, (M, K)).astype(np.float32)
        s = 2.0 ** rng.integers(-4, -1, (N, groups))
    else:
        x = rng.standard_normal((M, K)).astype(np.float32)
        s = rng.uniform(0.005, 0.02, (N, groups))
    z = rng.integers(0, 16, (N, groups)).astype(np.uint8) if zeros else None
    buf = torch.full((M, ldx or K), 7.0, dtype=_dtype(dtype), device=device)
    buf[:, :K] = torch.from_numpy(x)
    scales = torch.from_numpy(s).to(_dtype(dtype)).to(device)
    return dict(x=buf[:, :K], words=words, scales=scales, zeros=z, group=group,
                codes=torch.from_numpy(words.view(np.int32)).to(device),
                z=None if z is None else torch.from_numpy(z).to(device))


def _run(c, out_type, ldo=0, pack=None):
    import torch
    from ornith_g256 import native, storage
    N, K = c['words'].shape[0], c['words'].shape[1] * 8
    M = c['x'].shape[0]
    codes, meta = pack or storage.pack_w4(c['codes'], c['scales'], c['z'], c['group'])
    buf = torch.full((M, max(ldo, N)), -7.0, dtype=_dtype(out_type), device=c['x'].device)
    flags = torch.zeros(1, dtype=torch.int32, device=c['x'].device)
    native.w4_out(c['x'], codes, meta, buf[:, :N], flags, N, K, c['group'])
    torch.cuda.synchronize()
    assert bool((buf[:, N:] == -7.0).all())
    return buf[:, :N].double().cpu().numpy(), int(flags.item())


def _want(c):
    """(result, the sum of |s x| times 32) in float64."""
    s = c['scales'].double().cpu().numpy()
    x = c['x'].double().cpu().numpy()
    w = O.weights(c['words'], s, c['zeros'], c['group'])
    K = x.shape[1]
    return x @ w.T, 32 * np.abs(x) @ np.abs(s[:, np.arange(K) // c['group']]).T


def _check(c, got, out_type):
    want, scale = _want(c)
    K = c['x'].shape[1]
    steps = 128 + 3 + -(-K // 128) + 8
    tol = steps * 2.0 ** -23 * scale
    tol = tol + HALF_STEP[out_type] * (np.abs(want) + tol)
    if out_type == 'fp16':
        tol = tol + 2.0 ** -25                       # half a step of the subnormals
    bad = np.abs(got - want) > tol
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], tol[bad][:5])
    # the bound is loose by the square root of its length: the mean error is far below it
    ref = np.sqrt((want ** 2).mean())
    if ref > 0 and want.size > 64:
        assert np.sqrt(((got - want) ** 2).mean()) <= ref * (HALF_STEP[out_type] + 2.0 ** -20)


SHAPES = [(1, 1, 8), (1, 16, 32), (2, 15, 40), (1, 17, 128), (5, 100, 136), (16, 33, 256), (17, 64, 264),
          (33, 48, 520), (48, 30, 1024), (49, 257, 384), (64, 96, 2048), (65, 31, 640), (130, 40, 2120), (1, 2048, 512),
          (3, 1000, 4096), (8, 640, 8192), (1, 70000, 128), (7, 5003, 264), (3, 16, 32768), (2, 40, 65536)]


@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
@pytest.mark.parametrize('group', [32, 64, 128, 256])
@pytest.mark.parametrize('M,N,K', SHAPES)
def test_w4_whole_numbers(device, dtype, group, M, N, K):
    import torch
    print(f'w4 {dtype} group={group} M={M} N={N} K={K}', flush=True)
    rng = np.random.default_rng(M * 31 + N * 7 + K + group)
    zeros = bool((M + group // 32) % 2)
    c = _case(rng, M, N, K, group, zeros, dtype, device, True, ldx=K + 8 * (N % 3))
    got, flags = _run(c, 'fp32', ldo=N + N % 5)
    want, _ = _want(c)
    assert np.abs(want).max() < 2 ** 20 and flags == 0
    assert (got == want).all(), np.argwhere(got != want)[:5]
    got, flags = _run(c, dtype)
    assert (got == torch.from_numpy(want).to(_dtype(dtype)).double().numpy()).all()


@pytest.mark.parametrize('out_type', ['bf16', 'fp16', 'fp32'])
@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
@pytest.mark.parametrize('M,N,K', SHAPES)
def test_w4_rows(device, dtype, out_type, M, N, K):
    rng = np.random.default_rng(M + N + K)
    group = (32, 64, 128, 256)[(M + N) % 4]
    c = _case(rng, M, N, K, group, bool(N % 2), dtype, device, False)
    got, flags = _run(c, out_type)
    assert flags == 0
    _check(c, got, out_type)


# More than 16 rows of more than 3000 tiles of 16 x 16: x in shared memory, two, three and four tiles of
# rows a block, runs of columns that waves share in the middle of K and at its ends.
LONG = [(17, 24600, 8), (20, 25003, 2040), (32, 24592, 2048), (33, 16401, 1160), (40, 16400, 136), (48, 16500, 1304),
        (49, 12301, 1000), (64, 12320, 1024), (63, 12305, 2048), (130, 5500, 520), (200, 3801, 264)]


@pytest.mark.parametrize('group', [32, 64, 128, 256])
@pytest.mark.parametrize('M,N,K', LONG)
def test_w4_many_columns(device, group, M, N, K):
    import torch
    assert -(-N // 16) * -(-M // 16) > 3000
    rng = np.random.default_rng(M * 31 + N * 7 + K + group)
    dtype = ('bf16', 'fp16')[(M + group // 32) % 2]
    c = _case(rng, M, N, K, group, bool(K // 8 % 2), dtype, device, True, ldx=K + 8 * (N % 3))
    got, flags = _run(c, 'fp32', ldo=N + N % 5)
    want, _ = _want(c)
    assert np.abs(want).max() < 2 ** 20 and flags == 0
    assert (got == want).all(), np.argwhere(got != want)[:5]
    got, flags = _run(c, dtype)
    assert (got == torch.from_numpy(want).to(_dtype(dtype)).double().numpy()).all()


@pytest.mark.parametrize('out_type', ['bf16', 'fp16', 'fp32'])
@pytest.mark.parametrize('M,N,K', [(20, 25003, 2040), (33, 16401, 1160), (64, 12320, 1024)])
def test_w4_many_columns_rows(device, out_type, M, N, K):
    rng = np.random.default_rng(M + N + K)
    c = _case(rng, M, N, K, (32, 64, 128, 256)[M % 4], True, 'bf16' if M % 2 else 'fp16', device, False)
    got, flags = _run(c, out_type)
    assert flags == 0
    _check(c, got, out_type)
    c['x'][3] = float('nan')                           # raised from this kernel as well, and kept to its row
    some, flags = _run(c, out_type)
    assert flags == (4 if out_type == 'fp32' else 12)
    assert np.isnan(some[3]).all() and np.isfinite(np.delete(some, 3, 0)).all()


def test_pack_layout(device):
    import torch
    from ornith_g256 import storage
    rng = np.random.default_rng(3)
    for N, K, group, zeros in ((16, 128, 128, True), (37, 200, 32, True), (5, 8, 256, False), (64, 1000, 64, False)):
        for dtype in ('bf16', 'fp16'):
            c = _case(rng, 1, N, K, group, zeros, dtype, device, False)
            codes, meta = storage.pack_w4(c['codes'], c['scales'], c['z'], group)
            bits = c['scales'].float().cpu().numpy().view(np.uint32)
            wc, wm = O.packed(c['words'], bits, c['zeros'], group)
            assert (codes.cpu().numpy().view(np.uint32) == wc).all()
            assert (meta.cpu().numpy().view(np.uint32) == wm).all()


def test_a_row_does_not_depend_on_the_others(device):
    rng = np.random.default_rng(4)
    c = _case(rng, 64, 200, 1032, 64, True, 'bf16', device, False)
    full, _ = _run(c, 'fp32')
    c['x'][5] = float('nan')
    c['x'][40] = float('inf')
    some, flags = _run(c, 'fp32')
    rest = [m for m in range(64) if m not in (5, 40)]
    assert (some[rest] == full[rest]).all()
    assert np.isnan(some[5]).all() and not np.isfinite(some[40]).any()
    assert flags == 4


def test_flags(device):
    import torch
    rng = np.random.default_rng(5)
    c = _case(rng, 3, 40, 256, 128, False, 'fp16', device, True)
    c['x'][1] = 60000.0
    c['codes'].fill_(-1)                               # codes 15: sums of 256 * 60000 * 7 * s
    got, flags = _run(c, 'fp16')
    assert np.isinf(got[1]).all() and np.isfinite(got[[0, 2]]).all() and flags == 8
    got, flags = _run(c, 'fp32')
    assert np.isfinite(got).all() and flags == 0


def test_empty_calls(device):
    import torch
    from ornith_g256 import native, storage
    flags = torch.zeros(1, dtype=torch.int32, device=device)
    codes, meta = storage.pack_w4(torch.zeros((20, 4), dtype=torch.int32, device=device),
                                  torch.ones((20, 1), dtype=torch.bfloat16, device=device), None, 32)
    x = torch.zeros((0, 32), dtype=torch.bfloat16, device=device)
    native.w4_out(x, codes, meta, torch.empty((0, 20), dtype=torch.bfloat16, device=device), flags, 20, 32, 32)
    # no inputs: zeros
    codes, meta = storage.pack_w4(torch.zeros((20, 0), dtype=torch.int32, device=device),
                                  torch.ones((20, 0), dtype=torch.bfloat16, device=device), None, 32)
    out = torch.ones((3, 20), dtype=torch.float32, device=device)
    native.w4_out(torch.zeros((3, 0), dtype=torch.bfloat16, device=device), codes, meta, out, flags, 20, 0, 32)
    assert bool((out == 0).all()) and int(flags.item()) == 0
