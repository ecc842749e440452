"""Slices of an adapter call: none given is one part, an empty list is refused (no launch)."""
import pytest
import torch

from ornith_g256 import methods, native

BF = torch.bfloat16


@pytest.mark.parametrize('slices', [(), []])
def test_empty_slices(slices):
    args = dict(x=torch.zeros(3, 64, dtype=BF), a=torch.zeros(2, 8, 64, dtype=BF), b=torch.zeros(2, 40, 8, dtype=BF),
                scales=torch.ones(2), ids=torch.zeros(3, dtype=torch.int32), base=None, out=torch.zeros(3, 40, dtype=BF),
                workspace=torch.zeros(1 << 12, dtype=torch.uint8), flags=torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match='1 to 8 widths'):
        native.adapter_out(**args, slices=slices)
    with pytest.raises(ValueError, match='1 to 8 widths'):
        methods.LinearAdapters(40, 64, 2, 8, slices)
    with pytest.raises(ValueError, match='on one GPU'):                # (one part: refused for its place alone)
        native.adapter_out(**args, slices=None)
