"""Routing to experts against its definition in 64 bits.

Ids are compared exactly: the kernel's fp64 scores are within 2^-44 of
themselves and its picks within 2^-41, so rows whose oracle decisions are all
clearer than 2^-38 leave no choice; equal values go to the lowest id.  A weight
is rounded once to fp32: half a step, 2^-24, of itself, beside 2^-40 for the
scores and their sum (and half of fp32's smallest step, 2^-150)."""
import numpy as np
import pytest

from oracle import route as O

pytestmark = pytest.mark.gpu

CLEAR = 2.0 ** -38


def _dtype(name):
    import torch
    return {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}[name]


def _run(logits, top, score='softmax', bias=None, flags=None, **kw):
    import torch
    from ornith_g256 import native
    M, dev = logits.shape[0], logits.device
    weights = torch.full((M, top), 7.0, device=dev)
    ids = torch.full((M, top), 77, dtype=torch.int32, device=dev)
    flags = torch.zeros(1, dtype=torch.int32, device=dev)
    native.route_experts(logits, weights, ids, flags, score=score, bias=bias, **kw)
    torch.cuda.synchronize()
    return weights.cpu().numpy().astype(np.float64), ids.cpu().numpy(), int(flags)


def _check(logits, top, score='softmax', bias=None, groups=1, kept_groups=1, group_top=1, renormalize=True, scale=1.0,
           want_flags=0):
    w, ids, flags = _run(logits, top, score, bias, groups=groups, kept_groups=kept_groups, group_top=group_top,
                         renormalize=renormalize, scale=scale)
    host = logits.double().cpu().numpy()
    b = None if bias is None else bias.double().cpu().numpy()
    unclear = 0
    for m, row in enumerate(host):
        ww, wi, clear = O.route(row, top, score, b, groups, kept_groups, group_top, renormalize, scale)
        if clear < CLEAR:
            unclear += 1
            continue
        assert (ids[m] == wi).all(), (m, ids[m], wi, clear)
        tol = np.abs(ww) * (2.0 ** -24 + 2.0 ** -40) + 2.0 ** -150
        assert (np.abs(w[m] - ww) <= tol).all(), (m, w[m], ww)
    assert unclear <= 0.01 * len(host)
    assert flags == want_flags
    return w, ids


# experts, top, groups, kept groups
SHAPES = [(1, 1, 1, 1), (2, 2, 1, 1), (7, 3, 1, 1), (8, 2, 1, 1), (16, 4, 4, 2), (60, 4, 1, 1), (63, 32, 1, 1), (64, 6, 8, 3),
          (65, 8, 5, 2), (96, 6, 3, 1), (128, 8, 1, 1), (160, 6, 8, 3), (256, 8, 1, 1), (256, 8, 8, 4), (255, 8, 5, 4),
          (257, 9, 1, 1), (384, 8, 1, 1), (512, 10, 1, 1), (512, 22, 64, 5), (1000, 17, 40, 9), (1024, 32, 1, 1),
          (1023, 31, 33, 2), (992, 20, 32, 1), (64, 5, 64, 9)]


@pytest.mark.parametrize('dtype', ['bf16', 'fp16', 'fp32'])
@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('E,k,G,kept', SHAPES)
def test_route(device, dtype, score, E, k, G, kept):
    import torch
    print(f'route {dtype} {score} E={E} k={k} G={G} kept={kept}', flush=True)
    rng = np.random.default_rng(E * 5 + k + G)
    for rows, pad, biased, top2, renorm in ((1, 0, False, 1, True), (5, 3, True, 2, False), (70, 0, True, 1, True),
                                            (33, 1, False, 2, False)):
        buf = torch.full((rows, E + pad), float('nan'), dtype=_dtype(dtype), device=device)
        buf[:, :E] = torch.from_numpy(rng.standard_normal((rows, E)) * 2)
        bias = torch.from_numpy((rng.standard_normal(E) * 0.05).astype(np.float32)).to(device) if biased else None
        _check(buf[:, :E], k, score, bias, G, kept, top2, renorm, 2.5 if rows == 5 else 1.0)


@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('G,kept', [(1, 1), (8, 3)])
def test_ties_go_to_the_lowest_id(device, score, G, kept):
    import torch
    rng = np.random.default_rng(3)
    logits = torch.from_numpy(rng.integers(-2, 2, (200, 128)).astype(np.float32)).to(device)
    logits[7] = 0.0
    logits[8] = -0.0
    logits[9, ::2] = -0.0
    logits[9, 1::2] = 0.0
    # every two values of a row are equal or far apart, so every row is decided
    for bias in (None, torch.zeros(128, device=device)):
        w, ids = _check(logits, 8, score, bias, G, kept, 2)
        assert (ids[7] == np.arange(8)).all() and (ids[8] == np.arange(8)).all() and (ids[9] == np.arange(8)).all()


def test_masked_and_odd_rows(device):
    """-inf, NaN and the type's lowest values in the logits, a bias of -inf; rows with too few experts or none."""
    import torch
    inf = float('inf')
    for score in ('softmax', 'sigmoid'):
        base = torch.linspace(-3, 3, 64, device=device).repeat(9, 1)
        base[1, 8:] = -inf                             # exactly 8 left
        base[2, :60] = -inf                            # 4 left
        base[3] = -inf                                 # none
        base[4] = torch.finfo(torch.float32).min       # all at the lowest value: ties
        base[5, 5] = inf
        base[5, 9] = inf
        base[6, 1:] = torch.finfo(torch.float32).min
        base[7] = -1e30
        base[7, 20:40] = -500.0
        w, ids = _check(base, 8, score, want_flags=4)
        assert (ids[3] == -1).all() and (w[3] == 0).all()
        assert (ids[2, 4:] == -1).all() and (w[2, 4:] == 0).all() and abs(w[2].sum() - 1) < 1e-6
        assert (ids[4] == np.arange(8)).all() and np.isfinite(w).all()
        assert ids[5, 0] == 5 and ids[5, 1] == 9
        _check(base[[0, 1, 4, 5, 6, 7]], 8, score)
        _check(base, 8, score, groups=8, kept_groups=2, group_top=2, want_flags=4)
        _check(base, 8, score, renormalize=False, want_flags=4)
        bias = torch.zeros(64, device=device)
        bias[50:] = -inf
        _, ids = _check(base[[0, 4]], 8, score, bias)
        assert ids.max() < 50
        # logits that differ past where a sigmoid is 1, and where both scores are 0
        far = torch.tensor([[40.0, 60.0, 50.0, 90.0], [-800.0, -900.0, -1000.0, -850.0]], device=device)
        _, ids = _check(far, 3, score)
        assert ids.tolist() == [[3, 1, 2], [0, 3, 1]]
        nan = base[:1].clone()
        nan[0, 63] = float('nan')
        w, ids = _check(nan, 8, score, want_flags=1)
        assert 63 not in ids
        bad = torch.zeros(64, device=device)
        bad[3] = float('nan')
        w, ids, flags = _run(base[:1], 8, score, bad)
        assert flags == 1 and 3 not in ids and (ids >= 0).all()


def test_a_group_with_one_expert_left(device):
    """A group's score is of those that take part: one best where one is left, no score where none is."""
    import torch
    logits = torch.full((3, 16), -float('inf'), device=device)
    logits[0, [0, 4, 5, 8]] = torch.tensor([3.0, 1.0, 1.0, 0.5], device=device)
    logits[1, [15]] = 1.0
    logits[2, [2, 6, 7, 12]] = torch.tensor([-1.0, -5.0, -5.0, -0.9], device=device)
    for score in ('softmax', 'sigmoid'):
        for top2 in (1, 2):
            _check(logits, 4, score, groups=4, kept_groups=2, group_top=top2, want_flags=4)


def test_a_row_does_not_depend_on_the_others(device):
    import torch
    rng = np.random.default_rng(5)
    logits = torch.from_numpy(rng.standard_normal((300, 256)).astype(np.float32)).to(device)
    w, ids, _ = _run(logits, 8, groups=8, kept_groups=4)
    w1, ids1, _ = _run(logits[123:124], 8, groups=8, kept_groups=4)
    assert (w[123] == w1[0]).all() and (ids[123] == ids1[0]).all()


@pytest.mark.parametrize('bad', [dict(score='relu'), dict(groups=3), dict(groups=8, kept_groups=9), dict(kept_groups=0),
                                 dict(group_top=3), dict(scale=float('inf')), dict(scale=float('nan')), dict(scale=1e39),
                                 dict(groups=32, kept_groups=1)])
def test_refusals(device, bad):
    import torch
    from ornith_g256 import native
    z = torch.zeros((2, 64), device=device)
    out = torch.zeros((2, 4), device=device), torch.zeros((2, 4), dtype=torch.int32, device=device)
    flags = torch.zeros(1, dtype=torch.int32, device=device)
    with pytest.raises(ValueError):
        native.route_experts(z, *out, flags, **bad)
    native.route_experts(z[:0], out[0][:0], out[1][:0], flags)
    assert int(flags) == 0
