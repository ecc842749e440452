"""Plain 4-bit linears on both sides of every border at which another kernel is
taken, whole numbers bit for bit (test_gpu_w4)."""
import pytest

import test_gpu_w4 as G

pytestmark = pytest.mark.gpu


def _cells(M, N):
    return -(-M // 16) * -(-N // 16)


# three and four tiles of rows with x in shared memory: from 4097 tiles of results on
@pytest.mark.parametrize('group', [32, 64, 128, 256])
@pytest.mark.parametrize('M,N,K', [(33, 21841, 1280), (40, 22000, 136), (48, 21857, 1032), (49, 16385, 1000), (64, 16400, 1024),
                                   (63, 16390, 8), (130, 7300, 520), (200, 5100, 264), (64, 16384, 1024), (48, 21840, 512)])
def test_many_columns(device, group, M, N, K):
    assert _cells(M, N) > 4096 or (M, N) in ((64, 16384), (48, 21840))
    G.test_w4_many_columns(device, group, M, N, K)


# few rows or columns: one, two and four tiles of columns a block, 8 and 16 waves
@pytest.mark.parametrize('group', [32, 64, 128, 256])
@pytest.mark.parametrize('M,N,K', [(8, 4096, 1160), (3, 4090, 2048), (8, 4097, 2056), (1, 6143, 2184), (4, 6128, 2184), (2, 6144, 2048),
                                   (5, 6129, 1024), (4, 24577, 264), (5, 65530, 136), (8, 65521, 136), (16, 16384, 264),
                                   (16, 16385, 264), (33, 5461, 136), (12, 12273, 264), (20, 24000, 264), (20, 24001, 264),
                                   (17, 8192, 2056), (64, 2048, 4104)])
def test_tiles(device, group, M, N, K):
    G.test_w4_whole_numbers(device, ('bf16', 'fp16')[(N // 16 + group // 32) % 2], group, M, N, K)


# the rows of a prompt: many passes over the columns, and more of them than a grid's other axis has blocks for
@pytest.mark.parametrize('group', [32, 128])
@pytest.mark.parametrize('M,N,K', [(700, 1000, 520), (2100, 130, 264), (513, 2050, 2056), (16500, 60, 264), (9000, 17, 1544)])
def test_prompt_rows(device, group, M, N, K):
    G.test_w4_whole_numbers(device, 'bf16', group, M, N, K)
