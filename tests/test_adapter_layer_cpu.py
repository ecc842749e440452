"""Adapters beside a layer, and expert routing of a block: what they keep and
refuse (no launch)."""
import pytest
import torch

from ornith_g256 import methods, native

BF = torch.bfloat16


class _Layer(torch.nn.Module):
    def __init__(self, method):
        super().__init__()
        self.quant_method = method
        method.create_weights(self)


def _w4(n=48, k=64):
    return _Layer(methods.W4LinearMethod('lin', n, k))


def test_slots_are_padded_and_emptied():
    layer = _w4()
    ad = methods.attach_adapters(layer, slots=3, rank=16, slices=(16, 32))
    assert layer.adapters is ad and ad.a.shape == (3, 32, 64) and ad.b.shape == (3, 48, 16) and ad.scales.shape == (3,)
    a = [torch.randn(8, 64).to(BF), torch.randn(8, 64).to(BF)]
    b = torch.randn(48, 8).to(BF)
    ad.a.fill_(7)
    ad.b.fill_(7)
    ad.load(1, a, b, 0.5)
    assert torch.equal(ad.a[1, :8], a[0]) and torch.equal(ad.a[1, 16:24], a[1]) and torch.equal(ad.b[1, :, :8], b)
    assert not ad.a[1, 8:16].any() and not ad.a[1, 24:].any() and not ad.b[1, :, 8:].any() and float(ad.scales[1]) == 0.5
    assert bool((ad.a[0] == 7).all()) and bool((ad.b[2] == 7).all())
    ad.load(1, [None, a[1]], b)
    assert not ad.a[1, :16].any() and torch.equal(ad.a[1, 16:24], a[1]) and float(ad.scales[1]) == 1
    ad.drop(1)
    assert not ad.a[1].any() and not ad.b[1].any() and float(ad.scales[1]) == 0
    # not part of a checkpoint
    assert not any('adapters' in k for k in layer.state_dict())
    for bad in (dict(slot=3), dict(slot=-1), dict(a=a[0]), dict(a=a[:1]), dict(b=b[:40]), dict(b=b[:, :4]), dict(b=b[0]),
                dict(a=[a[0][:, :32], a[1]]), dict(a=[torch.zeros(24, 64)] * 2, b=torch.zeros(48, 24))):
        with pytest.raises(ValueError):
            ad.load(**(dict(slot=0, a=a, b=b) | bad))
    with pytest.raises(ValueError):
        ad.drop(3)


@pytest.mark.parametrize('bad', [dict(rank=12), dict(rank=0), dict(rank=520), dict(slots=0), dict(slots=4097), dict(slices=(40,)),
                                 dict(slices=(-1, 49)), dict(slices=(6,) * 8 + (0,)), dict(dtype=torch.float32)])
def test_banks_that_do_not_fit(bad):
    with pytest.raises(ValueError):
        methods.attach_adapters(_w4(), **(dict(slots=2, rank=8) | bad))


def test_where_adapters_go():
    head = _Layer.__new__(_Layer)
    torch.nn.Module.__init__(head)
    head.quant_method = methods.W8HeadMethod('head')
    for layer in (head, torch.nn.Linear(8, 8)):
        with pytest.raises(ValueError):
            methods.attach_adapters(layer, 2, 8)
    layer = _w4()
    layer.quant_method.runtime = object()
    with pytest.raises(RuntimeError):
        methods.attach_adapters(layer, 2, 8)
    g256 = _Layer(methods.G256LinearMethod('dense', 256, 512))
    assert methods.attach_adapters(g256, 2, 8).k == 512


def test_runtime_sizes_its_workspace_and_keeps_ids():
    native.reset_binding()
    try:
        plain = methods.Runtime(torch.nn.ModuleDict(dict(lin=_w4())), {}, 64, 'cpu')
        assert plain.adapter_ids is None
        with pytest.raises(RuntimeError):
            plain.set_adapter_ids(torch.zeros(3, dtype=torch.int32))
        layer = _w4(n=4096, k=64)
        methods.attach_adapters(layer, 2, 512)
        rt = methods.Runtime(torch.nn.ModuleDict(dict(lin=layer)), {}, 8192, 'cpu')
        assert rt.workspace.numel() >= native.adapter_bytes(8192, 512)
        assert rt.adapter_ids.shape == (8192,) and bool((rt.adapter_ids == -1).all())
        rt.set_adapter_ids(torch.tensor([1, 0, -1], dtype=torch.int32))
        rt.set_adapter_ids(torch.tensor([0, 1], dtype=torch.int32))
        assert rt.adapter_ids[:4].tolist() == [0, 1, -1, -1]
        for bad in (torch.zeros(8193, dtype=torch.int32), torch.zeros(3), torch.zeros((1, 3), dtype=torch.int32)):
            with pytest.raises(ValueError):
                rt.set_adapter_ids(bad)
        with pytest.raises(ValueError):
            layer.adapters.add(rt, torch.zeros(8193, 64, dtype=BF), torch.zeros(8193, 4096, dtype=BF), rt.slots[0])
    finally:
        native.reset_binding()


def test_routing_of_a_block(monkeypatch):
    seen = []
    monkeypatch.setattr(native, 'route_experts', lambda *a: seen.append(a))
    bias = torch.zeros(256)
    method = methods.G256MoEMethod('moe', methods.ExpertRouting(8, 'sigmoid', 8, 4, 2, True, 2.5, bias))
    with pytest.raises(RuntimeError):
        method.apply_logits(None, None, torch.zeros(3, 256))
    method.runtime, method.slot = type('Runtime', (), dict(slots=(torch.zeros(1, dtype=torch.int32),))), 0
    monkeypatch.setattr(method, 'apply', lambda layer, x, w, ids, **kw: (w.shape, w.dtype, ids.shape, ids.dtype))
    assert method.apply_logits(None, None, torch.zeros(3, 256)) == ((3, 8), torch.float32, (3, 8), torch.int32)
    assert seen[0][4:] == ('sigmoid', bias, 8, 4, 2, True, 2.5)
    with pytest.raises(ValueError):
        method.apply_logits(None, None, torch.zeros(3, 128))
    with pytest.raises(ValueError):
        methods.G256MoEMethod('moe', methods.ExpertRouting(6))
    assert methods.G256MoEMethod('moe').routing.score == 'softmax'


@pytest.mark.parametrize('name', ['gate_up_proj', 'down_proj'])
def test_no_adapters_on_a_shared_expert(name):
    """Its fused slot and fixed8 would not see them."""
    mlp = torch.nn.Module()
    for proj, n, k in (('gate_up_proj', 1024, 2048), ('down_proj', 2048, 512)):
        setattr(mlp, proj, _Layer(methods.G256LinearMethod(proj, n, k)))
    mlp.expert_gate = torch.nn.Linear(2048, 1, bias=False, dtype=BF)
    methods.SharedExpert('shared', mlp)
    methods.attach_adapters(getattr(mlp, name), 2, 8)
    with pytest.raises(ValueError, match='no adapters'):
        methods.SharedExpert('shared', mlp)
