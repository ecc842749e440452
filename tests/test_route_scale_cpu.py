"""The factor on routing weights: any finite fp32 number (no launch)."""
import pytest
import torch

from ornith_g256 import native


@pytest.mark.parametrize('scale,taken', [(torch.finfo(torch.float32).max, True), (-torch.finfo(torch.float32).max, True),
                                         (3.4028235e38, False), (-3.5e38, False), (0.0, True)])
def test_scale(scale, taken):
    with pytest.raises(ValueError, match='on one GPU' if taken else 'finite fp32'):
        native.route_experts(torch.zeros(3, 16), torch.zeros(3, 4), torch.zeros(3, 4, dtype=torch.int32),
                             torch.zeros(1, dtype=torch.int32), scale=scale)
