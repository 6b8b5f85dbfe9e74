"""Refusals of what shapes the chunk attention's scores, on the CPU."""
import numpy as np
import pytest
import torch

from dotcache_amd.chunk import attend_cached, attend_chunk, plan_chunk
from tests.test_chunk_cache_host import H, HD, HQ, _paged
from tests.test_chunk_host import _pools


def _call(**kw):
    kp, vp = _pools()
    plan = plan_chunk(kp, vp, [2], [20], kv_heads=2, q_per_kv=3)
    table = torch.zeros((1, 2, 2), dtype=torch.int32)
    return attend_chunk(kp, table, vp, table, torch.zeros((2, 6, 64)), plan, **kw)


@pytest.mark.parametrize("cap", [1e-46, 1e-60, np.float64(1e-46), 1e39, -1e-46])
def test_caps_that_fp32_does_not_hold(cap):
    """0 means no cap to the C entry, so one that rounds to 0 must not reach it."""
    with pytest.raises(ValueError, match="cap must be positive"):
        _call(cap=cap)


def test_caps_that_it_holds():
    for cap in (1e-45, 1e-30, 1, np.float32(2.5), 2e38):  # (these get as far as the tensors, which are on the CPU)
        with pytest.raises(ValueError, match="must be on a GPU"):
            _call(cap=cap)


@pytest.mark.parametrize("order", [None, [1, 0, 1, 0]])
@pytest.mark.parametrize("slopes", [torch.zeros(2 * HQ), torch.zeros(HQ - 1), torch.zeros(HQ, 2)[:, 0], torch.zeros(HQ, dtype=torch.float64),
                                    torch.zeros(1, HQ), torch.zeros(HQ, device="meta"), [0.0] * HQ, np.zeros(HQ, np.float32)])
def test_slopes_of_a_cache_are_checked_in_any_order_of_heads(slopes, order):
    cache = _paged()
    n = np.array([2], dtype=np.int32)
    table = torch.zeros((1, H, 1), dtype=torch.int32)
    default = np.repeat(np.arange(H), HQ // H)
    with pytest.raises(ValueError, match="slopes must be"):
        attend_cached(cache, torch.zeros((2, HQ, HD)), n, n, table, table, order, default, 1.0, slopes=slopes)
