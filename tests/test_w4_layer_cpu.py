"""The plain 4-bit layer method around its launch: what it keeps and what it
hands on."""
import weakref

import pytest
import torch

from ornith_g256 import methods, storage


class _Layer(torch.nn.Module):
    def __init__(self, n=48, k=64, **kw):
        super().__init__()
        self.quant_method = methods.W4LinearMethod('lin', n, k, **kw)
        self.quant_method.create_weights(self)


@pytest.mark.parametrize('zeros', [False, True])
def test_packing_drops_the_loaded_fields(monkeypatch, zeros):
    """Loaded where they are packed, codes, scales and zero points would take
    the banks' memory a second time."""
    seen = []

    def pack(codes, scales, zeros, group):
        seen.append((codes.shape, scales.shape, None if zeros is None else zeros.shape, group))
        return torch.zeros(3, 1, 64, 4, dtype=torch.int32), torch.zeros(3, 1, 16, 2, dtype=torch.int32)
    monkeypatch.setattr(storage, 'pack_w4', pack)
    layer = _Layer(group=64, zeros=zeros)
    fields = {'w4_codes': torch.zeros(48, 8, dtype=torch.int32).view(torch.uint32),
              'w4_scales': torch.ones(48, 1, dtype=torch.bfloat16)}
    if zeros:
        fields['w4_zeros'] = torch.full((48, 1), 8, dtype=torch.uint8)
    refs = []
    for name in list(fields):
        value = fields.pop(name)
        refs.append(weakref.ref(value.untyped_storage()))
        layer.load_packed(name, value)
        del value
    assert all(r() is not None for r in refs)
    layer.quant_method.process_weights_after_loading(layer)
    assert seen == [((48, 8), (48, 1), (48, 1) if zeros else None, 64)]
    assert all(r() is None for r in refs)
    assert not list(layer.parameters()) and {n for n, _ in layer.named_buffers()} == {'w4_bank', 'w4_metadata'}
    with pytest.raises(storage.AdmissionError):           # still sealed
        layer.load_packed('w4_codes', torch.zeros(48, 8, dtype=torch.int32).view(torch.uint32))


def _bound(**kw):
    layer = _Layer(**kw)
    layer.w4_bank = layer.w4_metadata = None
    method = layer.quant_method
    method.runtime, method.slot = type('Runtime', (), dict(slots=(torch.zeros(1, dtype=torch.int32),))), 0
    return layer


@pytest.mark.parametrize('lead,shape,strides', [(0, (3, 64), (64, 1)), (1, (3, 64), (64, 1)), (4, (1, 64), (64, 1)),
                                                (7, (2, 3, 64), (192, 64, 1)), (0, (3, 64), (68, 1)), (8, (3, 64), (72, 1)),
                                                (0, (5, 64), (1, 5)), (0, (3, 64), (0, 1)), (3, (0, 64), (64, 1))])
def test_rows_off_the_grid_are_copied(monkeypatch, lead, shape, strides):
    """The launch takes rows on the 16-byte grid; a contiguous view may start off
    it, where contiguous() copies nothing."""
    calls = []
    monkeypatch.setattr(methods.native, 'w4_out', lambda x, *a: calls.append(x))
    layer = _bound()
    buf = torch.arange(4096, dtype=torch.float32).to(torch.bfloat16)
    assert buf.data_ptr() % 16 == 0
    x = buf[lead:].as_strided(shape, strides)
    out = layer.quant_method.apply(layer, x)
    (rows,), want = calls, x.reshape(-1, 64)
    assert out.shape == (*shape[:-1], 48) and torch.equal(rows, want)
    if want.numel():
        assert rows.data_ptr() % 16 == 0 and rows.stride(1) == 1 and rows.stride(0) % 8 == 0
        # rows that are on it are not
        assert (rows.data_ptr() == x.data_ptr()) == (lead % 8 == 0 and strides[-1] == 1 and strides[-2] % 8 == 0 and strides[-2] >= 64)


def _compiled(fn, result):
    """fn under a full-graph compile whose graphs are kept and not run."""
    graphs = []

    def backend(graph, _):
        graphs.append(graph)
        return lambda *args: result
    torch._dynamo.reset()
    return torch.compile(fn, fullgraph=True, backend=backend), graphs


def _targets(graph):
    return [str(n.target) for n in graph.graph.nodes if n.op == 'call_function']


def test_the_layer_compiles():
    """As the G256 linears do: one op in the graph, no break."""
    layer = _bound()
    shapes = methods.native.w4_layout(48, 64, 128)
    layer.w4_bank, layer.w4_metadata = (torch.zeros(s, dtype=torch.int32) for s in shapes)
    run, graphs = _compiled(lambda x: layer.quant_method.apply(layer, x) * 2, (torch.zeros(3, 48),))
    run(torch.zeros(3, 64, dtype=torch.bfloat16))
    assert len(graphs) == 1 and 'ornith_g256.w4_out.default' in _targets(graphs[0])


@pytest.mark.parametrize('settings', [{}, dict(top_k=torch.ones(3, dtype=torch.int32)),
                                      dict(temperature=torch.ones(3), top_p=torch.ones(3), min_p=torch.zeros(3))])
def test_the_heads_sampler_compiles(settings):
    head = methods.W8HeadMethod('head')
    layer = torch.nn.Module()
    layer._ornith_loader = type('Loader', (), dict(sealed=True))
    layer.head_tilebank_codes = layer.head_scales = torch.zeros(1, dtype=torch.int32)
    head.runtime = type('Runtime', (), dict(slots=(torch.zeros(1, dtype=torch.int32),), head_geometry=2,
                                            workspace=torch.zeros(16, dtype=torch.uint8)))
    head.slot = 0
    run, graphs = _compiled(lambda x, u: head.sample(layer, x, u, **settings),
                            (torch.zeros(3, dtype=torch.int64), torch.zeros(3)))
    run(torch.zeros(3, 2048, dtype=torch.bfloat16), torch.zeros(3))
    names = _targets(graphs[0])
    assert len(graphs) == 1
    assert names.index('ornith_g256.head_out.default') < names.index('ornith_g256.logits_sample.default')


def test_dispatch_modes_see_the_ops():
    """Tracers that are not the compiler: fake tensors through the plain entries."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from ornith_g256 import native
    with FakeTensorMode():
        flags = torch.zeros(1, dtype=torch.int32)
        out = torch.empty(2, 48, dtype=torch.float32)
        shapes = native.w4_layout(48, 64, 128)
        native.w4_out(torch.zeros(2, 64, dtype=torch.bfloat16), *(torch.zeros(s, dtype=torch.int32) for s in shapes), out,
                      flags, 48, 64, 128)
        native.logits_sample(out, torch.zeros(2), torch.zeros(0, dtype=torch.uint8), torch.zeros(2, dtype=torch.int64), flags)
