"""Routing to experts: argument checks on the host (every case returns before a
launch), and the oracle against rows done by hand."""
import ctypes as C

import numpy as np
import pytest

from oracle import route as O

INVALID = 1


@pytest.fixture(scope='module')
def lib():
    from ornith_g256 import native
    return native.lib()


def _args(**kw):
    p = C.c_void_p
    a = dict(logits=p(0x10000), kind=2, M=2, E=64, ld=64, bias=p(0x20000), score=0, G=8, Gk=4, group_top=2, k=8, renorm=1,
             scale=1.0, weights=p(0x30000), ids=p(0x40000), flags=p(0x50000), stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize('bad', [dict(kind=3), dict(kind=-1), dict(M=-1), dict(E=0), dict(E=1025, ld=1025, G=1, Gk=1), dict(ld=63),
                                 dict(G=0), dict(G=7), dict(E=130, ld=130, G=65), dict(Gk=0), dict(Gk=9), dict(group_top=0),
                                 dict(group_top=3), dict(k=0), dict(k=33), dict(Gk=1, k=9), dict(score=2), dict(score=-1),
                                 dict(renorm=2), dict(scale=float('nan')), dict(scale=float('inf')), dict(logits=None),
                                 dict(weights=None), dict(ids=None), dict(flags=None), dict(logits=C.c_void_p(0x10002)),
                                 dict(bias=C.c_void_p(0x20002)), dict(weights=C.c_void_p(0x30001)),
                                 dict(ids=C.c_void_p(0x30020)), dict(flags=C.c_void_p(0x40004)),
                                 dict(weights=C.c_void_p(0x10004)), dict(ld=1 << 62)])
def test_launch_refusals(lib, bad):
    assert lib.ornith_route_experts_launch(*_args(**bad)) == INVALID


def test_nothing_to_do(lib):
    assert lib.ornith_route_experts_launch(*_args(M=0, logits=None, weights=None, ids=None, flags=None)) == 0


def test_python_refusals():
    import torch
    from ornith_g256 import native
    z = torch.zeros((3, 16))
    good = dict(logits=z, weights=torch.zeros(3, 4), ids=torch.zeros(3, 4, dtype=torch.int32),
                flags=torch.zeros(1, dtype=torch.int32))
    for bad in (dict(logits=z.double()), dict(logits=z[0]), dict(logits=z.t().contiguous().t()),
                dict(logits=z[:1].expand(3, 16)), dict(weights=torch.zeros(3, 5)), dict(weights=torch.zeros(3)),
                dict(weights=torch.zeros(3, 8)[:, ::2]), dict(ids=torch.zeros(3, 4, dtype=torch.int64)),
                dict(bias=torch.zeros(15)), dict(bias=torch.zeros(16, dtype=torch.bfloat16)), dict(score='top'),
                dict(flags=torch.zeros(2, dtype=torch.int32)), dict(weights=torch.zeros(3, 0), ids=torch.zeros(3, 0, dtype=torch.int32)),
                dict()):
        with pytest.raises(ValueError):
            native.route_experts(**(good | bad))


def test_oracle_by_hand():
    l = [0.0, np.log(2), np.log(4), -np.inf]
    w, ids, clear = O.route(l, 2)
    assert ids.tolist() == [2, 1] and np.allclose(w, [2 / 3, 1 / 3]) and clear > 0.4
    w, ids, _ = O.route(l, 2, renormalize=False, scale=7)
    assert np.allclose(w, [4, 2])
    w, ids, _ = O.route(l, 4, 'sigmoid', renormalize=False)
    assert ids.tolist() == [2, 1, 0, -1] and np.allclose(w, [0.8, 2 / 3, 0.5, 0])
    # a bias turns the pick and not the weights
    w, ids, _ = O.route(l, 2, 'sigmoid', bias=[1, 0, 0, 9], renormalize=False)
    assert ids.tolist() == [0, 2] and np.allclose(w, [0.5, 0.8])
    # groups (0, 1) and (2, 3): by one best the second, by two the first
    g = [0.0, 0.0, 0.5, -9.0]
    assert O.route(g, 2, 'sigmoid', groups=2, kept=1)[1].tolist() == [2, 3]
    assert O.route(g, 2, 'sigmoid', groups=2, kept=1, group_top=2)[1].tolist() == [0, 1]
    assert O.route([1.0, 1.0, 1.0], 2)[1].tolist() == [0, 1]
    assert O.route([-np.inf] * 3, 2)[1].tolist() == [-1, -1]
