"""Plain 4-bit linears: argument checks on the host (every case returns before
a launch) and the packed layout's round trip."""
import ctypes as C

import numpy as np
import pytest

from oracle import w4 as O

INVALID = 1


@pytest.fixture(scope='module')
def lib():
    from ornith_g256 import native
    return native.lib()


def test_layout(lib):
    from ornith_g256 import native
    c, m = C.c_size_t(0), C.c_size_t(0)
    q = lib.ornith_w4_get_layout
    for n, k, g in ((1, 8, 32), (17, 136, 64), (6144, 2048, 128), (0, 0, 256), (1 << 20, 8, 32)):
        assert q(n, k, g, C.byref(c), C.byref(m)) == 0
        shapes = native.w4_layout(n, k, g)
        assert c.value == np.prod(shapes[0]) and m.value == np.prod(shapes[1])
    for bad in ((-1, 8, 32), ((1 << 20) + 1, 8, 32), (1, 9, 32), (1, -8, 32), (1, 65544, 32), (1, 8, 48), (1, 8, 0)):
        assert q(*bad, C.byref(c), C.byref(m)) == INVALID
        with pytest.raises(RuntimeError):
            native.w4_layout(*bad)
    assert q(1, 8, 32, None, C.byref(m)) == INVALID


def _args(**kw):
    p = C.c_void_p
    a = dict(x=p(0x10000), x_type=0, ldx=256, codes=p(0x20000), meta=p(0x40000), out=p(0x50000), out_type=2, ldo=100,
             flags=p(0x60000), M=2, N=100, K=256, G=128, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize('bad', [dict(x_type=2), dict(x_type=-1), dict(out_type=3), dict(out_type=-1), dict(ldx=248),
                                 dict(ldx=260), dict(ldo=99), dict(M=-1), dict(N=-1), dict(K=250, ldx=256), dict(G=100),
                                 dict(x=None), dict(codes=None), dict(meta=None), dict(out=None), dict(flags=None),
                                 dict(x=C.c_void_p(0x10008)), dict(codes=C.c_void_p(0x20004)),
                                 dict(out=C.c_void_p(0x50002)), dict(meta=C.c_void_p(0x40002)),
                                 dict(out=C.c_void_p(0x10100)), dict(flags=C.c_void_p(0x50010)),
                                 dict(out=C.c_void_p(0x20100))])
def test_launch_refusals(lib, bad):
    assert lib.ornith_w4_launch(*_args(**bad)) == INVALID


def test_nothing_to_do(lib):
    assert lib.ornith_w4_launch(*_args(M=0)) == 0
    assert lib.ornith_w4_launch(None, 0, 8, None, None, None, 0, 0, None, 0, 0, 8, 32, None) == 0
    assert lib.ornith_w4_pack(None, None, 0, None, None, None, None, 0, 8, 32, None) == 0


@pytest.mark.parametrize('bad', [dict(t=2), dict(N=-1), dict(K=12), dict(G=16), dict(codes=None), dict(scales=None),
                                 dict(pc=None), dict(pm=None), dict(pc=C.c_void_p(0x40008)),
                                 dict(pm=C.c_void_p(0x40100)), dict(pc=C.c_void_p(0x10100)), dict(flags=None),
                                 dict(flags=C.c_void_p(0x80000))])
def test_pack_refusals(lib, bad):
    p = C.c_void_p
    a = dict(codes=p(0x10000), scales=p(0x20000), t=0, z=p(0x30000), pc=p(0x40000), pm=p(0x80000), flags=p(0x90000), N=40, K=256, G=64,
             stream=None) | bad
    assert lib.ornith_w4_pack(*a.values()) == INVALID


def test_python_refusals():
    import torch
    from ornith_g256 import native, storage
    x = torch.zeros(2, 32, dtype=torch.bfloat16)
    lay = native.w4_layout(20, 32, 32)
    codes, meta = torch.zeros(lay[0], dtype=torch.int32), torch.zeros(lay[1], dtype=torch.int32)
    out, flags = torch.zeros(2, 20, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    good = dict(x=x, codes=codes, metadata=meta, out=out, flags=flags, n=20, k=32, group=32)
    wide = torch.zeros(2, 36, dtype=torch.bfloat16)
    for bad in (dict(x=x.float()), dict(x=x[0]), dict(k=24), dict(out=out[:1]), dict(out=out.double()),
                dict(x=wide[:, :32]), dict(x=x.t().contiguous().t()), dict(x=x[:1].expand(2, 32)),
                dict(out=out[:1].expand(2, 20)), dict(codes=codes[:1]), dict(codes=codes.long()),
                dict(metadata=meta.transpose(0, 1)), dict(flags=flags.long()), dict(n=21), dict()):
        with pytest.raises(ValueError):
            native.w4_out(**(good | bad))
    with pytest.raises(ValueError):
        storage.pack_w4(torch.zeros(20, 4, dtype=torch.int32), torch.zeros(20, 1, dtype=torch.bfloat16), None, 32)


def test_packed_layout_by_hand():
    # column 3's k = 5 of the first block: lane 16 * 0 + 3, word 0, odd k: bits 16 + 4 * 2
    words = np.zeros((4, 16), np.uint32)
    words[3, 0] = 9 << 20
    bits = np.full((4, 1), 0x3f800000, np.uint32)
    codes, meta = O.packed(words, bits, None, 128)
    assert codes.shape == (1, 1, 64, 4) and meta.shape == (1, 1, 16, 1)
    assert codes[0, 0, 3, 0] == 9 << 24 and codes[0, 0, 3, 1] == 0
    assert codes[0, 0, 4, 0] == 0x88888888               # past N
    assert meta[0, 0, 3, 0] == 0x3f800008 and meta[0, 0, 4, 0] == 8
