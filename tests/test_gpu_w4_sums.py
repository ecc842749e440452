"""What the sums through 16 + c cost: rows with a mean, columns whose codes are
their zero point, and the largest rows that cannot overflow on the way.

A result is off by at most (128 + K / 128 + 11) 2^-23 of 32 sum |s x| before its
rounding to the output's type (test_gpu_w4's count of the additions): an
absolute error, also where the sum itself is 0."""
import numpy as np
import pytest

import test_gpu_w4 as G

pytestmark = pytest.mark.gpu

# (both kernels: x from memory, and more than 16 rows of many columns)
SHAPES = [(1, 2048, 512), (5, 100, 136), (8, 640, 8192), (64, 96, 2048), (20, 25003, 2040), (33, 16401, 1160)]


def _make(rng, M, N, K, group, dtype, device, x, codes, zeros, scales):
    import torch
    words = (codes.reshape(N, K // 8, 8).astype(np.uint32) << (4 * np.arange(8, dtype=np.uint32))).sum(2, dtype=np.uint32)
    return dict(x=torch.from_numpy(x).to(G._dtype(dtype)).to(device), words=words, group=group, zeros=zeros,
                scales=torch.from_numpy(scales).to(G._dtype(dtype)).to(device),
                codes=torch.from_numpy(words.view(np.int32)).to(device), z=torch.from_numpy(zeros).to(device))


@pytest.mark.parametrize('group', [32, 64, 128, 256])
@pytest.mark.parametrize('mean', [0.0, 5.0])
@pytest.mark.parametrize('M,N,K', SHAPES)
def test_means_and_pruned_columns(device, group, mean, M, N, K):
    rng = np.random.default_rng(M + N + K + group)
    dtype = ('bf16', 'fp16')[(M + group // 32) % 2]
    groups = -(-K // group)
    codes = rng.integers(0, 16, (N, K), dtype=np.uint8)
    zeros = rng.integers(0, 16, (N, groups)).astype(np.uint8)
    pruned = np.arange(N) % 3 == 1                     # codes equal to their zero points: the result is 0
    codes[pruned] = zeros[pruned][:, np.arange(K) // group]
    x = (mean + rng.standard_normal((M, K))).astype(np.float32)
    c = _make(rng, M, N, K, group, dtype, device, x, codes, zeros, rng.uniform(0.005, 0.02, (N, groups)))
    got, flags = G._run(c, 'fp32')
    want, scale = G._want(c)
    assert flags == 0 and (want[:, pruned] == 0).all()
    tol = (128 + 3 + -(-K // 128) + 8) * 2.0 ** -23 * scale
    tol = tol + 2.0 ** -24 * (np.abs(want) + tol)
    off = np.abs(got - want)
    print(f'{dtype} mean {mean} group {group} {M}x{N}x{K}: off by up to {(off / scale).max() * 2 ** 24:.3f} 2^-24 of 32 sum |s x|, '
          f'rms {np.sqrt(((off / scale) ** 2).mean()) * 2 ** 24:.3f}', flush=True)
    assert (off <= tol).all()


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
