"""Sampling: argument checks on the host (every case returns before a launch)
and the 64-bit definition on small rows worked by hand."""
import ctypes as C

import numpy as np
import pytest

from oracle import sampling as S

INVALID = 1


@pytest.fixture(scope='module')
def lib():
    from ornith_g256 import native
    return native.lib()


def test_layout(lib):
    from ornith_g256 import native
    size = C.c_size_t(0)
    q = lib.ornith_logits_sample_get_layout
    assert q(64, 248320, C.byref(size)) == 0 and size.value > 0
    assert q(0, 10000, C.byref(size)) == 0 and size.value == 0
    assert q(1, 1 << 20, C.byref(size)) == 0
    for bad in ((-1, 10), (1, -1), (1, (1 << 20) + 1)):
        assert q(*bad, C.byref(size)) == INVALID
    assert q(1, 10, None) == INVALID
    # rows of up to 8192 columns need none; many rows share what some use
    assert native.logits_sample_bytes(64, 8192) == 0 < native.logits_sample_bytes(1, 8193)
    assert native.logits_sample_bytes(1024, 10000) == native.logits_sample_bytes(4000, 10000)
    assert native.logits_sample_bytes(64, 248320) == native.logits_sample_bytes(65, 248320)
    assert native.logits_sample_bytes(2, 10000) < native.logits_sample_bytes(3, 10000)


def _args(**kw):
    p = C.c_void_p
    a = dict(logits=p(0x10000), type=0, M=2, N=10000, ld=10000, uniform=p(0x20000), T=p(0x21000), k=p(0x22000),
             p=p(0x23000), q=p(0x24000), ws=p(0x1000000), bytes=1 << 22, token=p(0x30000), logprob=p(0x31000),
             flags=p(0x32000), stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize('bad', [dict(type=3), dict(type=-1), dict(M=-1), dict(N=-1), dict(N=(1 << 20) + 1, ld=1 << 21),
                                 dict(ld=9999), dict(bytes=1000), dict(logits=None), dict(uniform=None),
                                 dict(token=None), dict(flags=None), dict(ws=None), dict(logits=C.c_void_p(0x10001)),
                                 dict(type=2, logits=C.c_void_p(0x10002)), dict(uniform=C.c_void_p(0x20002)),
                                 dict(token=C.c_void_p(0x30004)), dict(ws=C.c_void_p(0x1000080)),
                                 dict(T=C.c_void_p(0x30000)),           # a setting inside the tokens
                                 dict(flags=C.c_void_p(0x10010)),       # the flag word inside the logits
                                 dict(logprob=C.c_void_p(0x1000100))])  # the result inside the workspace
def test_refusals(lib, bad):
    assert lib.ornith_logits_sample_launch(*_args(**bad)) == INVALID


def test_no_rows_touch_nothing(lib):
    assert lib.ornith_logits_sample_launch(*_args(M=0)) == 0
    assert lib.ornith_logits_sample_launch(None, 0, 0, 5, 5, *[None] * 6, 0, *[None] * 4) == 0


def test_python_refusals():
    import torch
    from ornith_g256 import native
    x = torch.zeros(2, 8, dtype=torch.bfloat16)
    u, out, flags = torch.zeros(2), torch.zeros(2, dtype=torch.int64), torch.zeros(1, dtype=torch.int32)
    ws = torch.zeros(16, dtype=torch.uint8)
    for bad in (dict(logits=x.double()), dict(logits=x.t()), dict(logits=x[0]), dict(uniform=u.double()),
                dict(uniform=None), dict(uniform=torch.zeros(3)), dict(out=out.int()), dict(top_k=out),
                dict(temperature=torch.zeros(4)[::2]), dict(min_p=u.half()), dict(top_p=u.unsqueeze(1)),
                dict(logprob=u.double()), dict(flags=torch.zeros(2, dtype=torch.int32)),
                dict(logits=x[:1].expand(2, 8)), dict()):           # the last: not on a GPU
        args = dict(logits=x, uniform=u, workspace=ws, out=out, flags=flags) | bad
        with pytest.raises(ValueError):
            native.logits_sample(**args)


def test_definition_by_hand():
    row = np.log(np.array([1.0, 8.0, 4.0, 2.0, 1.0]))          # masses 1/8 1 1/2 1/4 1/8
    assert S.kept(row, 1.0)[0].tolist() == [0, 1, 2, 3, 4]
    assert S.kept(row, 1.0, k=4)[0].tolist() == [0, 1, 2, 3]     # the first of the equal ones
    assert S.kept(row, 1.0, p=0.51)[0].tolist() == [1, 2]
    assert S.kept(row, 1.0, k=2, p=0.6)[0].tolist() == [1]       # of the first two: 2 / 3
    assert S.kept(row, 1.0, q=0.24)[0].tolist() == [1, 2, 3]
    assert S.kept(row, 0.5, q=0.24)[0].tolist() == [1, 2]
    tok, lp = S.sample(row, 1.0, u=0.1)
    assert tok == 1 and abs(lp - np.log(0.5)) < 1e-12            # running: 1 9 13 15 16 of 16
    assert [S.sample(row, 1.0, u=v)[0] for v in (0.0, 0.05, 0.57, 0.9, 0.99)] == [0, 0, 2, 3, 4]
    assert S.sample(row, 0.0) == (1, 0.0)
    assert S.sample(np.full(3, -np.inf), 1.0)[0] == -1
