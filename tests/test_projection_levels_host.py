"""Which codes and levels a 4-bit weight takes, on the CPU."""
import numpy as np
import pytest
import torch

from dotcache_amd.projection import GroupedWeight


def _parts(scale, bias, N=20, K=40):
    full = lambda x: None if x is None else torch.full((N, 2), x).half()  # noqa: E731
    return torch.arange(N * K).reshape(N, K) % 15, full(scale), full(bias)


@pytest.mark.parametrize("scale,bias", [(8700.0, -65504.0), (-8700.0, 65504.0), (5000.0, -20000.0), (9352.0, None), (-9352.0, None), (0.0, 65504.0)])
def test_levels_in_range_are_taken(scale, bias):
    codes, s, b = _parts(scale, bias)
    dense = GroupedWeight.from_codes(codes, s, b, group_size=32).dense()
    want = codes.double() * float(s[0, 0]) + float(b[0, 0]) if bias is not None else (codes.double() - 7) * float(s[0, 0])
    assert torch.equal(dense.double(), want)


@pytest.mark.parametrize("scale,bias", [(8800.0, -65504.0), (-8800.0, 65504.0), (5000.0, -8000.0), (9376.0, None), (float("inf"), None),
                                        (float("nan"), 0.0), (1.0, float("inf")), (float("inf"), -float("inf"))])
def test_levels_out_of_range_are_refused(scale, bias):
    codes, s, b = _parts(scale, bias)
    with pytest.raises(ValueError, match="range"):
        GroupedWeight.from_codes(codes, s, b, group_size=32)


@pytest.mark.parametrize("dtype,code", [(torch.int64, 2 ** 32 + 5), (torch.int64, -2 ** 32 + 5), (torch.int64, 2 ** 40), (torch.uint32, 2 ** 32 - 1),
                                        (torch.uint32, 2 ** 31), (torch.uint64, 2 ** 32 + 5), (torch.uint64, 2 ** 63 + 5), (torch.int8, -1),
                                        (torch.uint8, 255), (torch.int32, 16)])
@pytest.mark.parametrize("affine", [True, False])
def test_codes_that_wrap_into_the_range_are_refused(dtype, code, affine):
    _, s, b = _parts(1.0, 0.0 if affine else None)
    codes = np.zeros((20, 40), dtype=str(dtype).split(".")[1])
    codes[19, 39] = code
    with pytest.raises(ValueError, match="codes must lie"):
        GroupedWeight.from_codes(torch.from_numpy(codes), s, b, group_size=32)
    codes[19, 39] = 14
    assert float(GroupedWeight.from_codes(torch.from_numpy(codes), s, b, group_size=32).dense()[19, 39]) == (14 if affine else 7)
