"""Adapters on both sides of each choice of a launch: rows with and without a plan,
one launch and two, 16 and 64 rows of A a block."""
import numpy as np
import pytest

import test_gpu_adapter as A

pytestmark = pytest.mark.gpu

# rows, columns, inputs, rank, slots, slices
SHAPES = [(M, N, 136, R, 5, parts) for R, parts in ((16, 1), (40, 2), (64, 1), (72, 1), (128, 2))
          for M, N in ((64, 1500), (65, 1500), (160, 4096), (160, 4097), (161, 4096), (256, 2560), (256, 2561), (256, 5120), (256, 5121),
                       (257, 500))]


@pytest.mark.parametrize('dtype', ['bf16', 'fp16'])
@pytest.mark.parametrize('M,N,K,R,slots,parts', SHAPES)
def test_whole_numbers(device, dtype, M, N, K, R, slots, parts):
    print(f'adapter {dtype} M={M} N={N} R={R}', flush=True)
    rng = np.random.default_rng(M + N + R)
    ids = np.sort(rng.integers(-1, slots, M)) if N % 2 else None       # runs of a request, or any
    c = A._case(rng, M, N, K, R, slots, parts, dtype, 'fp32' if M % 2 else dtype, device, True, ids=ids)
    A._check(c, A._run(c), exact=True)
    A._check(c, A._run(c, in_place=True), exact=True)


@pytest.mark.parametrize('M', [1, 8, 9, 32, 33, 64])
@pytest.mark.parametrize('R,parts', [(32, 1), (40, 1), (64, 2), (72, 1), (256, 1)])
def test_few_rows(device, M, R, parts):
    rng = np.random.default_rng(M + R)
    c = A._case(rng, M, 300, 2056, R, 7, parts, 'bf16', 'fp32', device, False)
    A._check(c, A._run(c))
