"""How much of an fp32 number its cut into 16-bit numbers holds, over every mantissa of
a binade: each number the rounding of what is left (include/ornith_adapter.h)."""
import pytest
import torch


def _left(v, dtype, parts):
    for _ in range(parts):
        v = v - v.to(dtype).float()                    # (exact: the rounding and the number are within a factor of two, or 0)
    return v


@pytest.mark.parametrize('dtype,parts,bound', [(torch.bfloat16, 2, 2.0 ** -17), (torch.bfloat16, 3, 0.0), (torch.float16, 2, 2.0 ** -23)])
def test_all_mantissas(dtype, parts, bound):
    at = 2.0 ** 14                                     # (where a row's largest is brought to in fp16)
    worst = 0.0
    for chunk in torch.arange(2 ** 23, dtype=torch.int32).split(2 ** 20):
        v = ((127 + 14 << 23) + chunk).view(torch.float32)
        worst = max(worst, float((_left(v, dtype, parts).abs() / v).max()))
        assert float((_left(v, dtype, parts).abs() / at).max()) <= bound
    assert bound / 2 < worst <= bound or worst == bound == 0.0


def test_three_parts_hold_small_numbers():
    """Down to 2^-103 the last of 24 bits is a normal bf16 number."""
    for e in (-103, -60, 0, 100):
        v = ((127 + e << 23) + torch.arange(0, 2 ** 23, 101, dtype=torch.int32)).view(torch.float32)
        assert not bool(_left(v, torch.bfloat16, 3).any())
        third = _left(v, torch.bfloat16, 2)
        assert float(third[third != 0].abs().min()) >= 2.0 ** -126
