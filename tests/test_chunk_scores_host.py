"""Refusals of what shapes the chunk attention's scores, on the CPU."""
import numpy as np
import pytest
import torch

from dotcache_amd.chunk import attend_chunk, plan_chunk
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
