"""The sums through 16 + c: the largest rows that cannot overflow on the way."""
import numpy as np
import pytest

import test_gpu_w4 as G

pytestmark = pytest.mark.gpu


def _make(rng, M, N, K, group, dtype, device, x, codes, zeros, scales):
    import torch
    words = (codes.reshape(N, K // 8, 8).astype(np.uint32) << (4 * np.arange(8, dtype=np.uint32))).sum(2, dtype=np.uint32)
    return dict(x=torch.from_numpy(x).to(G._dtype(dtype)).to(device), words=words, group=group, zeros=zeros,
                scales=torch.from_numpy(scales).to(G._dtype(dtype)).to(device),
                codes=torch.from_numpy(words.view(np.int32)).to(device), z=torch.from_numpy(zeros).to(device))


@pytest.mark.parametrize('group', [32, 64, 128, 256])
@pytest.mark.parametrize('M,N,K', [(3, 70, 1024), (20, 24600, 512)])
def test_largest_rows(device, group, M, N, K):
    """bf16 rows of one sign just below 2^116: 31 * 128 of them stay below 2^128.
    Their units are 2^108, at most 31 * 255 * 128 (a block of 128) and
    15 * 255 * K (the total) of them, below 2^24: every sum is exact."""
    rng = np.random.default_rng(group)
    groups = K // group
    x = np.full((M, K), 255 * 2.0 ** 108, np.float32)
    x[1] = -x[1]
    x[2, ::2] = -x[2, ::2]
    # columns of the largest sums, of the smallest, and of codes equal to their zero points
    codes = np.empty((N, K), np.uint8)
    zeros = np.empty((N, groups), np.uint8)
    for i, (code, zero) in enumerate(((15, 0), (0, 15), (8, 8), (15, 15), (0, 0))):
        codes[i::5], zeros[i::5] = code, zero
    c = _make(rng, M, N, K, group, 'bf16', device, x, codes, zeros, np.full((N, groups), 2.0 ** -20))
    got, flags = G._run(c, 'fp32')
    want, _ = G._want(c)
    assert flags == 0 and (got == want).all()
    got, flags = G._run(c, 'bf16')
    assert flags == 0 and (np.abs(got - want) <= 2.0 ** -8 * np.abs(want)).all()
