"""Which rows a layer's adapters are taken for: the step's, or those that the call
names (no launch)."""
import pytest
import torch

from ornith_g256 import methods, native

BF = torch.bfloat16


class _Layer(torch.nn.Module):
    def __init__(self, method):
        super().__init__()
        self.quant_method = method
        method.create_weights(self)


@pytest.fixture
def seen(monkeypatch):
    """ids of each addition, in place of the launches."""
    calls = []
    monkeypatch.setattr(native, 'w4_out', lambda *a: None)
    monkeypatch.setattr(native, 'dense_out', lambda *a: None)
    monkeypatch.setattr(native, 'adapter_out', lambda x, a, b, scales, ids, base, out, ws, flags, slices: calls.append(ids.tolist()))
    native.reset_binding()
    yield calls
    native.reset_binding()


def _w4(out_dtype=None, adapters=True, **kw):
    layer = _Layer(methods.W4LinearMethod('lin', 48, 64, out_dtype=out_dtype))
    layer.w4_bank = layer.w4_metadata = None
    if adapters:
        methods.attach_adapters(layer, 4, 8, **kw)
    return layer


def _g256(**kw):
    layer = _Layer(methods.G256LinearMethod('dense', 256, 512))
    layer._ornith_loader.sealed = True
    methods.attach_adapters(layer, 4, 8, **kw)
    return layer


def _bind(**layers):
    return methods.Runtime(torch.nn.ModuleDict(layers), {}, 64, 'cpu')


def _call(layer, rows, **kw):
    return layer.quant_method.apply(layer, torch.zeros(rows, layer.quant_method.k, dtype=BF), **kw)


IDS = torch.tensor([3, 2, 1, 0, -1, 3, 1, 2], dtype=torch.int32)


@pytest.mark.parametrize('make', [_w4, _g256])
def test_rows_of_a_step(seen, make):
    layer = make()
    rt = _bind(lin=layer)
    _call(layer, 5)
    rt.set_adapter_ids(IDS)
    _call(layer, 8)
    _call(layer, 10)                                   # a padded batch: no adapters past the step's rows
    assert seen == [[-1] * 5, IDS.tolist(), IDS.tolist() + [-1, -1]]
    # fewer rows than the step has could be any of them
    with pytest.raises(ValueError, match='adapter_ids'):
        _call(layer, 3)
    assert _call(layer, 0).shape[0] == 0
    _call(layer, 3, adapter_ids=IDS[[4, 0, 7]])
    assert seen[3:] == [[], [-1, 3, 2]]
    rt.set_adapter_ids(IDS[:2])
    _call(layer, 3)
    assert seen[5:] == [[3, 2, -1]]


def test_a_head_names_its_rows(seen):
    head, declared, plain = _w4(torch.float32), _w4(step_rows=False), _w4(torch.float32, step_rows=True)
    rt = _bind(head=head, declared=declared, plain=plain)
    assert (head.adapters.step_rows, declared.adapters.step_rows, plain.adapters.step_rows) == (False, False, True)
    rt.set_adapter_ids(IDS)
    for layer in (head, declared):
        for rows in (3, 8):
            with pytest.raises(ValueError, match='adapter_ids'):
                _call(layer, rows)
        _call(layer, 2, adapter_ids=IDS[[1, 6]])
    _call(plain, 8)
    assert seen == [[2, 1], [2, 1], IDS.tolist()]


def test_ids_without_adapters_are_refused(seen):
    layer = _w4(adapters=False)
    _bind(lin=layer)
    assert _call(layer, 3).shape == (3, 48)
    with pytest.raises(ValueError, match='without adapters'):
        _call(layer, 3, adapter_ids=IDS[:3])
    assert seen == []
