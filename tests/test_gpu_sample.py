"""Sampling against its definition in 64 bits.

A uniform number is placed in the middle of the chosen token's interval and a
top-p in the middle of its prefix's, so both are decided by arithmetic: the
kernels' masses are off by half a unit of 2^-36 of their part's power of two
(at most twice the part's largest mass), by 2^-33 of themselves (polynomial)
and by |t| 2^-53 (argument), so a running sum of n masses relative to the
largest is off by at most n 2^-36 + S 2^-32; fp32 u and p are off by 2^-25.
Intervals narrower than MARGIN of the kept mass, eight times fp32's step, are
not chosen, and n 2^-36 stays below that for the n used here.
logprob: fp32 of ln(e / S): half a step of the result, and the masses' errors
relative to S, below 2^-21 + 2^-25 in all."""
import numpy as np
import pytest

from oracle import sampling as S

pytestmark = pytest.mark.gpu

MARGIN = 2.0 ** -21
PART, LIST_LDS, LIST_MAX = 8192, 8192, 16384


def _np(t):
    return t.double().cpu().numpy()


def _run(logits, u, T=None, k=None, p=None, q=None, workspace_fill=None):
    import torch
    from ornith_g256 import native
    M, N = logits.shape
    dev = logits.device
    ws = torch.empty(native.logits_sample_bytes(M, N), dtype=torch.uint8, device=dev)
    if workspace_fill is not None:
        ws.fill_(workspace_fill)
    token = torch.full((M,), -7, dtype=torch.int64, device=dev)
    logprob = torch.full((M,), 7.0, device=dev)
    flags = torch.zeros(1, dtype=torch.int32, device=dev)

    def dev_t(v, dtype):
        return None if v is None else torch.as_tensor(np.asarray(v), dtype=dtype).to(dev)
    native.logits_sample(logits, dev_t(u, torch.float32), ws, token, flags, dev_t(T, torch.float32),
                         dev_t(k, torch.int32), dev_t(p, torch.float32), dev_t(q, torch.float32), logprob)
    torch.cuda.synchronize()
    return token.cpu().numpy(), logprob.double().cpu().numpy(), int(flags.item())


def _logits(rng, M, N, dtype, device, lead=0, pad=0, scale=2.0):
    import torch
    buf = torch.zeros(lead + M * (N + pad), dtype=dtype, device=device)
    view = buf[lead:].view(M, N + pad)[:, :N]
    view.copy_(torch.from_numpy((rng.standard_normal((M, N)) * scale).astype(np.float32)))
    return view


def _dtype(name):
    import torch
    return {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}[name]


def _place(rng, row, T, k, p, q):
    """A uniform number for a random kept token whose interval is wide enough."""
    cols, e = S.kept(row, T, k, p, q)
    wide = cols[e >= 2 * MARGIN * e.sum()]
    col = int(rng.choice(wide))
    u, width = S.uniform_for(row, T, k, p, q, col)
    return np.float32(u), col


def _settings(rng, row, which):
    T = float(np.float32(rng.choice([0.3, 0.7, 1.0, 1.5])))
    k, p, q = 0, 1.0, 0.0
    n = len(S.order(row))
    if 'k' in which:
        k = int(rng.integers(1, min(n, 300) + 1))
    if 'p' in which:
        e = S.masses(row, S.order(row), T)[:k or n]
        ok = np.flatnonzero(e >= 2 * MARGIN * e.sum())
        p = float(np.float32(S.top_p_for(row, T, k, int(rng.choice(ok)) + 1)[0]))
        if not 0 < p < 1:
            p = 1.0
    if 'q' in which:
        q = float(np.float32(rng.uniform(0.001, 0.5)))
    return T, k, p, q


def _check(logits, Ts, ks, ps, qs, us, want=None, **kw):
    rows = _np(logits)
    token, logprob, flags = _run(logits, us, Ts, ks, ps, qs, **kw)
    for m, row in enumerate(rows):
        tok, lp = S.sample(row, Ts[m], ks[m], float(np.float32(ps[m])), float(np.float32(qs[m])), float(us[m]))
        assert token[m] == tok, (m, token[m], tok, Ts[m], ks[m], ps[m], qs[m], us[m])
        if want is not None:
            assert tok == want[m]
        assert abs(logprob[m] - lp) <= 2.0 ** -24 * abs(lp) + 2.0 ** -21, (m, logprob[m], lp)
    assert flags == 0


@pytest.mark.parametrize('dtype', ['bf16', 'fp16', 'fp32'])
@pytest.mark.parametrize('M,N,lead,pad', [(1, 1, 0, 0), (2, 2, 1, 0), (3, 7, 3, 2), (5, 64, 0, 1), (4, 1000, 0, 0),
                                          (3, PART - 1, 1, 0), (3, PART, 0, 0), (3, PART + 1, 0, 5),
                                          (2, 2 * PART + 1, 7, 3), (3, 50001, 0, 7), (1, 151936, 0, 0),
                                          (2, 248320, 0, 8), (70, 600, 0, 0)])
@pytest.mark.parametrize('which', ['', 'k', 'p', 'q', 'kp', 'kpq'])
def test_sample_shapes(device, dtype, M, N, lead, pad, which):
    print(f'sample {dtype} M={M} N={N} lead={lead} pad={pad} which={which}', flush=True)
    rng = np.random.default_rng(M * 1000003 + N * 7 + len(which))
    logits = _logits(rng, M, N, _dtype(dtype), device, lead, pad)
    rows = _np(logits)
    Ts, ks, ps, qs, us, cols = [], [], [], [], [], []
    for row in rows:
        T, k, p, q = _settings(rng, row, which)
        u, col = _place(rng, row, T, k, p, q)
        for l, v in zip((Ts, ks, ps, qs, us, cols), (T, k, p, q, u, col)):
            l.append(v)
    _check(logits, Ts, ks, ps, qs, us, cols, workspace_fill=0xff)


def test_settings_off_and_null_agree(device):
    """A NULL setting is the setting's off value."""
    import torch
    rng = np.random.default_rng(5)
    logits = _logits(rng, 6, 20000, torch.bfloat16, device)
    us = rng.random(6).astype(np.float32)
    a = _run(logits, us)
    b = _run(logits, us, [1.0] * 6, [0] * 6, [1.0] * 6, [0.0] * 6)
    c = _run(logits, us, [1.0] * 6, [20000] * 6, [1.0] * 6, [1e-30] * 6)
    for x in (b, c):
        assert (a[0] == x[0]).all() and (a[1] == x[1]).all() and x[2] == 0


def test_a_row_does_not_depend_on_the_others(device):
    import torch
    rng = np.random.default_rng(6)
    logits = _logits(rng, 67, 30000, torch.bfloat16, device)
    us = rng.random(67).astype(np.float32)
    T, k = rng.uniform(0.2, 1.5, 67), rng.integers(0, 100, 67)
    p, q = rng.uniform(0.5, 1, 67), rng.uniform(0, 0.05, 67)
    tok, lp, _ = _run(logits, us, T, k, p, q)
    for m in (0, 13, 63, 64, 66):
        t1, l1, _ = _run(logits[m:m + 1], us[m:m + 1], T[m:m + 1], k[m:m + 1], p[m:m + 1], q[m:m + 1])
        assert t1[0] == tok[m] and l1[0] == lp[m]


@pytest.mark.parametrize('N', [5, 5000, 20000, 50001, 270000])
@pytest.mark.parametrize('value', [0.0, -3.4028234663852886e38, 3.0e38, np.inf])
def test_equal_logits(device, N, value):
    """Every mass is the same: cuts and draws are decided by whole numbers.  From
    a list in shared memory over one in global memory to none."""
    import torch
    logits = torch.full((6, N), value, dtype=torch.float32, device=device)
    if value == 0.0:
        logits[:, ::3] = -0.0                          # equal to +0
    half = N // 2
    u = (np.array([0, 0, 0.5, 0.5, 0.25, 0.75]) + 0.25 / N).astype(np.float32)
    k = [0, 1, half, 0, half, 0]
    p = [1.0, 1.0, 1.0, 0.5, 0.5, 0.25]
    q = [0.0, 0.0, 0.0, 1.0, 0.0, 0.5]
    token, logprob, flags = _run(logits, u, [1.0, 0.5, 1.0, 2.0, 1e-3, 1e6], k, p, q)
    for m in range(6):
        n = k[m] or N
        n = int(np.ceil(n * p[m]))
        assert token[m] == int(np.floor(float(u[m]) * n)), (m, token[m], n)
        assert abs(logprob[m] + np.log(n)) <= 2.0 ** -24 * np.log(max(n, 2)) + 2.0 ** -21
    assert flags == 0


def test_ties_take_the_lowest_columns(device):
    """A border inside a run of equal values, on columns of several parts."""
    import torch
    rng = np.random.default_rng(8)
    N = 40000
    logits = torch.full((4, N), -4.0, dtype=torch.bfloat16, device=device)
    ties = np.sort(rng.choice(N, 60, replace=False))
    logits[:, torch.from_numpy(ties).to(device)] = 2.0
    logits[:, N - 3] = 3.0
    rows = _np(logits)
    ties = ties[ties != N - 3]
    for n in (2, 31, len(ties)):
        # the n-th value of the order is the (n - 1)-th tie: draw it, the last one kept
        last = int(ties[n - 2])
        us, ps = [], []
        for m, row in enumerate(rows):
            p = np.float32(S.top_p_for(row, 0.5, 0, n)[0]) if m % 2 else np.float32(1)
            kq = (0 if m % 2 else n)
            us.append(np.float32(S.uniform_for(row, 0.5, kq, float(p), 0.0, last)[0]))
            ps.append(p)
        _check(logits, [0.5] * 4, [0 if m % 2 else n for m in range(4)], ps, [0.0] * 4, us, [last] * 4)


def test_masked_rows(device):
    import torch
    rng = np.random.default_rng(9)
    N = 30000
    logits = _logits(rng, 8, N, torch.float32, device)
    low = float(np.finfo(np.float32).min)
    logits[0] = -np.inf                                # nothing
    logits[1] = -np.inf
    logits[1, 29999] = -5.0                            # one
    logits[2] = low                                    # masks of the type's lowest value
    logits[2, 12345] = 1.0
    logits[3, :] = low                                 # nothing but those
    logits[4, 100:29000] = -np.inf
    logits[5, 8192:16384] = -np.inf                    # a whole part
    logits[6, 17] = np.nan
    logits[6, 20000:20050] = np.nan
    logits[7] = np.nan
    us = np.full(8, 0.5 + 2.0 ** -20, np.float32)
    T, k, p, q = [1.0] * 8, [0, 0, 5, 0, 40, 0, 3, 0], [0.9] * 8, [0.0] * 8
    token, logprob, flags = _run(logits, us, T, k, p, q)
    assert token[0] == -1 and np.isnan(logprob[0]) and token[7] == -1 and np.isnan(logprob[7])
    assert token[1] == 29999 and logprob[1] == 0
    assert token[2] == 12345 and abs(logprob[2]) <= 2.0 ** -21
    rows = _np(logits)
    for m in (3, 4, 5, 6):
        tok, lp = S.sample(rows[m], 1.0, k[m], float(np.float32(0.9)), 0.0, float(us[m]))
        assert token[m] == tok and abs(logprob[m] - lp) <= 2.0 ** -24 * abs(lp) + 2.0 ** -21, m
    assert flags == 1 | 4


def test_greedy_rows_follow_argmax(device):
    import torch
    from ornith_g256 import native
    rng = np.random.default_rng(10)
    logits = _logits(rng, 5, 70001, torch.bfloat16, device)
    logits[1, 50000] = logits[1].max()
    logits[2] = -0.0
    logits[2, 5] = 0.0
    logits[3, 60000] = np.inf
    want = torch.empty(5, dtype=torch.int64, device=device)
    native.logits_argmax(logits.contiguous(), want)
    token, logprob, flags = _run(logits, [0.7] * 5, [0.0] * 5, [5] * 5, [0.1] * 5, [0.5] * 5)
    w = want.cpu().numpy()
    assert (token[[0, 1, 3, 4]] == w[[0, 1, 3, 4]]).all() and token[2] == 0
    assert (logprob == 0).all() and flags == 0


def test_infinite_logits_share_the_draw(device):
    import torch
    logits = torch.zeros((3, 20000), dtype=torch.float32, device=device)
    logits[:, [7, 9000, 19999]] = np.inf
    token, logprob, flags = _run(logits, [0.1, 0.5, 0.9], [1.0, 0.5, 2.0], [0, 3, 0], [1.0, 1.0, 0.9], [0, 0, 0.5])
    assert token.tolist() == [7, 9000, 19999] and flags == 0
    assert np.abs(logprob + np.log(3)).max() <= 2.0 ** -23


@pytest.mark.parametrize('name,bad', [('T', -1.0), ('T', np.nan), ('T', np.inf), ('p', 0.0), ('p', 1.5), ('p', np.nan),
                                      ('q', -0.1), ('q', 1.5), ('u', 1.0), ('u', -0.5), ('u', np.nan)])
def test_settings_out_of_range_raise_the_flag(device, name, bad):
    import torch
    rng = np.random.default_rng(11)
    logits = _logits(rng, 3, 9000, torch.float16, device)
    v = dict(T=[0.8] * 3, p=[0.9] * 3, q=[0.01] * 3, u=[0.3] * 3, k=[50] * 3)
    good = _run(logits, v['u'], v['T'], v['k'], v['p'], v['q'])
    v[name][1] = bad
    token, logprob, flags = _run(logits, v['u'], v['T'], v['k'], v['p'], v['q'])
    assert flags == 2 and token[1] == -1 and np.isnan(logprob[1])
    assert (token[[0, 2]] == good[0][[0, 2]]).all() and (logprob[[0, 2]] == good[1][[0, 2]]).all()


@pytest.mark.parametrize('T', [1e-30, 1e-3, 30.0, 1e4, 3e38])
def test_extreme_temperatures(device, T):
    import torch
    rng = np.random.default_rng(12)
    logits = _logits(rng, 4, 12000, torch.float32, device)
    T = float(np.float32(T))
    rows = _np(logits)
    ks, qs = [0, 100, 0, 50], [0.0, 0.0, 0.5, 0.0]
    us = [_place(rng, row, T, k, 1.0, q)[0] for row, k, q in zip(rows, ks, qs)]
    _check(logits, [T] * 4, ks, [1.0] * 4, qs, us)


def test_uniform_ends(device):
    import torch
    rng = np.random.default_rng(13)
    logits = _logits(rng, 4, 10000, torch.float32, device, scale=1.0)
    rows = _np(logits)
    last = np.float32(1 - 2.0 ** -24)
    token, _, flags = _run(logits, [0.0, 0.0, last, last], [1.0] * 4, [0, 7, 3, 1], [1.0] * 4, [0.0] * 4)
    for m, k in ((0, 0), (1, 7)):
        assert token[m] == S.kept(rows[m], 1.0, k)[0][0]
    for m, k in ((2, 3), (3, 1)):
        assert token[m] == S.kept(rows[m], 1.0, k)[0][-1]
    assert flags == 0


@pytest.mark.parametrize('N', [PART + 1, LIST_LDS + LIST_LDS // 2, LIST_MAX, LIST_MAX + 1])
@pytest.mark.parametrize('levels', [1, 2, 40])
def test_border_lists_of_every_length(device, N, levels):
    """All values in one bin: border lists in shared memory, past it, and rows
    that have none.  The levels differ by 2^-10 in t, less than a bin's eighth;
    every kept mass is above 2^-14.2 of the sum, so each interval is wide enough."""
    import torch
    rng = np.random.default_rng(N + levels)
    step = 2.0 ** -10 * np.log(2.0)
    logits = torch.from_numpy((rng.integers(0, levels, (5, N)) * -step).astype(np.float32)).to(device)
    rows = _np(logits)
    ks = [0, 1 + N // 3, N - 1, 0, N // 2]
    ps = [np.float32(S.top_p_for(row, 1.0, k, n)[0]) for row, k, n in
          zip(rows, ks, (N // 5, N // 4, N - 7, N // 2 + 1, 3))]
    us, cols = zip(*[_place(rng, row, 1.0, k, float(p), 0.0) for row, k, p in zip(rows, ks, ps)])
    _check(logits, [1.0] * 5, ks, ps, [0.0] * 5, us, cols)


@pytest.mark.parametrize('dtype', ['bf16', 'fp32'])
@pytest.mark.parametrize('N', [600, 10000, 40000])
@pytest.mark.parametrize('sign', [1, -1])
def test_sorted_rows(device, dtype, N, sign):
    """The largest values side by side at one end, and top-k about its bounds."""
    import torch
    rng = np.random.default_rng(N + sign)
    ks = [1, 2, 63, 64, 65, 255, 256, 257, 300, 500]
    base = np.sort(rng.standard_normal((len(ks), N)) * 2, axis=1)[:, ::sign]
    logits = torch.from_numpy(base.astype(np.float32)).to(_dtype(dtype)).to(device)
    rows = _np(logits)
    us, cols = zip(*[_place(rng, row, 1.0, k, 1.0, 0.0) for row, k in zip(rows, ks)])
    _check(logits, [1.0] * len(ks), ks, [1.0] * len(ks), [0.0] * len(ks), us, cols)


@pytest.mark.parametrize('dtype', ['bf16', 'fp32'])
@pytest.mark.parametrize('M', [1, 2, 3])
@pytest.mark.parametrize('which', ['', 'k', 'p', 'kpq'])
def test_longest_rows(device, dtype, M, which):
    """2^20 columns.  Off by half a unit of 2^-36 of at most twice the largest
    mass each, n masses are off by 2^-16 of the largest together: 2^-22 of
    a sum of 64 of it or more, within MARGIN."""
    rng = np.random.default_rng(M * 31 + len(which))
    N = 1 << 20
    logits = _logits(rng, M, N, _dtype(dtype), device, lead=1)
    settings = []
    for row in _np(logits):
        T, k, p, q = _settings(rng, row, which)
        T = max(T, 1.0)
        if 'p' in which:                               # (of the T that is used)
            p = float(np.float32(S.top_p_for(row, T, k, 2 + int(rng.integers(0, 20)))[0]))
        if not k:
            assert S.masses(row, S.order(row), T).sum() >= 64
        u, col = _place(rng, row, T, k, p, q)
        settings.append((T, k, p, q, u, col))
    Ts, ks, ps, qs, us, cols = zip(*settings)
    _check(logits, Ts, ks, ps, qs, us, cols, workspace_fill=0xff)


@pytest.mark.parametrize('M,N', [(530, 9000), (70, 130000)])
def test_rows_past_a_chunk(device, M, N):
    """More rows than one pass takes: as if each part of them were alone."""
    import torch
    from ornith_g256 import native
    rng = np.random.default_rng(M)
    assert native.logits_sample_bytes(M, N) == native.logits_sample_bytes(2 * M, N)
    logits = _logits(rng, M, N, torch.bfloat16, device)
    us = rng.random(M).astype(np.float32)
    T, k = rng.choice([0.0, 0.5, 1.0], M), rng.choice([0, 1, 50, 2000], M)
    p, q = rng.choice([1.0, 0.9, 0.3], M), rng.choice([0.0, 0.1], M)
    token, logprob, flags = _run(logits, us, T, k, p, q)
    for r in range(0, M, 60):
        s = slice(r, r + 60)
        t1, l1, f1 = _run(logits[s], us[s], T[s], k[s], p[s], q[s])
        assert (t1 == token[s]).all() and (l1 == logprob[s]).all() and f1 == 0, r
    assert flags == 0


@pytest.mark.parametrize('dtype', ['bf16', 'fp16', 'fp32'])
def test_every_launch_plan_agrees(device, dtype):
    """Rows of every kind with every cut: few parts at a time (two launches), all
    at once (four), and in one block, give the same bits."""
    import torch
    rng = np.random.default_rng(15)
    N = 40000
    top = float(torch.finfo(_dtype(dtype)).max)
    kinds = rng.standard_normal((12, N)).astype(np.float32) * 2
    kinds[1] = 0.0
    kinds[2] = -np.inf
    kinds[3] = -np.inf
    kinds[3, 33333] = -4.0
    kinds[4] = -top
    kinds[4, 77] = 2.0
    kinds[5, 5::7] = np.nan
    kinds[6, [3, 9000, 39999]] = np.inf
    kinds[7] = np.linspace(-20, 20, N)
    kinds[8] = top
    kinds[8, ::2] = -top
    kinds[9, 8192:16384] = -np.inf
    kinds[10, rng.random(N) > 0.02] = -np.inf
    kinds[11] = rng.integers(0, 2, N)
    cuts = [(0, 1.0, 0.0, 1.0), (1, 1.0, 0.0, 1.0), (50, 0.9, 0.0, 0.7), (0, 0.95, 0.0, 1.0), (0, 1.0, 0.05, 0.8),
            (300, 1.0, 0.0, 1.5), (20000, 0.5, 1e-6, 1.0), (39999, 0.999, 0.0, 100.0), (40, 0.9, 0.1, 0.0),
            (5, 0.9, 0.0, -1.0)]
    logits = torch.from_numpy(kinds).to(_dtype(dtype)).to(device).repeat(len(cuts), 1)
    us = rng.random(12 * len(cuts)).astype(np.float32)
    k, p, q, T = (np.repeat([c[i] for c in cuts], 12) for i in range(4))
    token, logprob, flags = _run(logits, us, T, k, p, q)
    assert len(us) * 5 > 256 and flags == 7
    for r in range(0, len(us), 12):
        s = slice(r, r + 12)
        t1, l1, _ = _run(logits[s], us[s], T[s], k[s], p[s], q[s])
        assert (t1 == token[s]).all() and np.array_equal(l1, logprob[s], equal_nan=True), (cuts[r // 12], t1, token[s])
    # rows of one part: their end is masked, and then it is not there
    masked = logits.clone()
    masked[:, PART:] = -float('inf')
    token, logprob, _ = _run(masked, us, T, k, p, q)
    t1, l1, _ = _run(masked[:, :PART].contiguous(), us, T, k, p, q)
    same = (k < PART) | (p < 1)                        # (with a top-k past all that is there, that is all)
    assert (t1 == token)[same].all() and np.array_equal(l1[same], logprob[same], equal_nan=True)
