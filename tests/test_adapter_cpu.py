"""Adapters: argument checks on the host (every case returns before a launch)."""
import ctypes as C

import pytest

INVALID = 1


@pytest.fixture(scope='module')
def lib():
    from ornith_g256 import native
    return native.lib()


def _args(**kw):
    p = C.c_void_p
    a = dict(x=p(0x100000), x_type=0, ldx=256, a=p(0x200000), a_slot=2 * 16 * 256, b=p(0x300000), b_slot=100 * 16,
             scales=p(0x400000), ids=p(0x410000), base=p(0x500000), ldb=100, out=p(0x600000), out_type=0, ldo=104,
             ws=p(0x700000), ws_bytes=1 << 20, flags=p(0x900000), M=5, N=100, K=256, R=16, S=2,
             ends=(C.c_int * 2)(40, 100), slots=3, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return list(a.values())


def _ends(*v):
    return (C.c_int * len(v))(*v)


@pytest.mark.parametrize('bad', [
    dict(x_type=2), dict(x_type=-1), dict(out_type=3), dict(out_type=-1), dict(ldx=248), dict(ldx=260), dict(ldb=99), dict(ldo=99),
    dict(a_slot=2 * 16 * 256 - 8), dict(a_slot=2 * 16 * 256 + 4), dict(b_slot=1592), dict(b_slot=1604), dict(M=-1), dict(N=-1),
    dict(N=(1 << 20) + 1), dict(K=250), dict(K=65544, ldx=65544, a_slot=1 << 24), dict(K=-8), dict(R=12), dict(R=0), dict(R=520),
    dict(S=0), dict(S=9), dict(slots=-1), dict(slots=4097), dict(ends=None), dict(ends=_ends(40, 99)), dict(ends=_ends(101, 100)),
    dict(ends=_ends(-1, 100)), dict(x=None), dict(a=None), dict(b=None), dict(scales=None), dict(ids=None), dict(base=None),
    dict(out=None), dict(ws=None), dict(flags=None), dict(ws_bytes=64), dict(x=C.c_void_p(0x100008)),
    dict(a=C.c_void_p(0x200008)), dict(b=C.c_void_p(0x300008)), dict(out=C.c_void_p(0x600001)), dict(base=C.c_void_p(0x500001)),
    dict(ids=C.c_void_p(0x410002)), dict(scales=C.c_void_p(0x400002)), dict(ws=C.c_void_p(0x700010)),
    dict(out=C.c_void_p(0x500010)), dict(out=C.c_void_p(0x100100)), dict(out=C.c_void_p(0x700100)),
    dict(out=C.c_void_p(0x500000)), dict(flags=C.c_void_p(0x600000)), dict(ldx=1 << 61), dict(ldo=1 << 61), dict(a_slot=1 << 61)])
def test_launch_refusals(lib, bad):
    # (out on base with another row stride is refused; with the same one it is an addition in place)
    assert lib.ornith_adapter_launch(*_args(**bad)) == INVALID


def test_nothing_to_do(lib):
    assert lib.ornith_adapter_launch(*_args(M=0)) == 0
    assert lib.ornith_adapter_launch(*_args(N=0, ends=_ends(0, 0), out=None)) == 0


def test_layout(lib):
    from ornith_g256 import native
    size = C.c_size_t(0)
    for m, s, r in ((0, 1, 8), (1, 1, 16), (64, 3, 64), (8192, 8, 512), (1 << 24, 1, 8)):
        assert lib.ornith_adapter_get_layout(m, s, r, C.byref(size)) == 0
        rows = min(m, 1 << 20)
        assert size.value >= rows * (s * r * 4 + 4)
        assert native.adapter_bytes(m, s * r) == size.value
    # what a capacity has room for, every smaller batch has, however its rows of A are divided
    for rows_of_a, ways in ((64, ((1, 64), (8, 8), (2, 32))), (512, ((1, 512), (8, 64), (2, 256))), (192, ((3, 64), (1, 192)))):
        last = 0
        for m in (0, 1, 63, 64, 65, 255, 256, 257, 1000, 1023, 1024, 4095, 4096, 8192, 1 << 20, (1 << 20) + 1):
            sizes = set()
            for s, r in ways:
                assert lib.ornith_adapter_get_layout(m, s, r, C.byref(size)) == 0
                sizes.add(size.value)
            assert len(sizes) == 1 and size.value >= last
            last = size.value
    for bad in ((-1, 1, 8), (1, 0, 8), (1, 9, 8), (1, 1, 4), (1, 1, 12), (1, 1, 520)):
        assert lib.ornith_adapter_get_layout(*bad, C.byref(size)) == INVALID
    assert lib.ornith_adapter_get_layout(1, 1, 8, None) == INVALID
    for bad in (0, 12, 8 * 521 * 8):
        with pytest.raises((ValueError, RuntimeError)):
            native.adapter_bytes(1, bad)


def test_python_refusals():
    import torch
    from ornith_g256 import native
    bf = torch.bfloat16
    x, a, b = torch.zeros(3, 64, dtype=bf), torch.zeros(2, 16, 64, dtype=bf), torch.zeros(2, 40, 8, dtype=bf)
    out = torch.zeros(3, 40, dtype=bf)
    good = dict(x=x, a=a, b=b, scales=torch.ones(2), ids=torch.zeros(3, dtype=torch.int32), base=out.clone(), out=out,
                workspace=torch.zeros(1 << 12, dtype=torch.uint8), flags=torch.zeros(1, dtype=torch.int32), slices=(10, 30))
    wide = torch.zeros(3, 68, dtype=bf)
    for bad in (dict(x=x.float()), dict(x=x[0]), dict(x=x[:, :56]), dict(x=wide[:, :64]), dict(x=x[:1].expand(3, 64)),
                dict(x=x.t().contiguous().t()), dict(a=a.half()), dict(a=a[:1]), dict(a=a[:, :8]), dict(a=a.transpose(1, 2)),
                dict(a=a.transpose(0, 1).contiguous().transpose(0, 1)), dict(b=b.float()), dict(b=b[:, :, :4]),
                dict(b=b.transpose(0, 1).contiguous().transpose(0, 1)), dict(slices=(10, 20)), dict(slices=None),
                dict(slices=(-10, 50)), dict(slices=(5,) * 8 + (0,)), dict(out=out.double()), dict(out=out[:2]),
                dict(out=out[:1].expand(3, 40)), dict(base=out.float()), dict(base=out[:2]), dict(base=out[:1].expand(3, 40)),
                dict(ids=None), dict(ids=torch.zeros(3, dtype=torch.int64)), dict(ids=torch.zeros(2, dtype=torch.int32)),
                dict(scales=None), dict(scales=torch.ones(3)), dict(scales=torch.ones(2, dtype=bf)),
                dict(flags=torch.zeros(1)), dict(workspace=torch.zeros(64)), dict()):
        with pytest.raises(ValueError):
            native.adapter_out(**(good | bad))
