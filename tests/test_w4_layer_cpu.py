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
