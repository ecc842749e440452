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


@pytest.mark.parametrize('lead,ldo', [(0, 208), (0, 203), (3, 208)])
@pytest.mark.parametrize('M,R,out_type', [(300, 72, 'bf16'), (1100, 128, 'fp32'), (4200, 96, 'fp16'), (300, 16, 'bf16'), (4200, 64, 'fp32')])
def test_results_on_and_off_the_grid(device, M, R, out_type, lead, ldo):
    """Rows of results that start on 16 bytes or not, what lies between them as it was."""
    import torch
    from ornith_g256 import native
    c = A._case(np.random.default_rng(M + R), M, 200, 136, R, 3, 1, 'bf16', out_type, device, True)
    buf = torch.full((lead + M * ldo,), -7.0, dtype=c['base'].dtype, device=device)
    assert buf.data_ptr() % 16 == 0
    out = buf[lead:].view(M, ldo)[:, :200]
    flags = torch.zeros(1, dtype=torch.int32, device=device)
    ws = torch.full((native.adapter_bytes(M, R),), 0xff, dtype=torch.uint8, device=device)
    native.adapter_out(c['x'], c['a'], c['b'], c['scales'], c['ids'], c['base'], out, ws, flags)
    A._check(c, (out, int(flags)), exact=True)
    assert bool((buf[:lead] == -7).all()) and bool((buf[lead:].view(M, ldo)[:, 200:] == -7).all())
