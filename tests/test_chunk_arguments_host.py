"""Arguments of the chunk attention that are refused before any launch
(pointers here are never read)."""
import pytest
import torch

from dotcache_amd import _lib
from dotcache_amd.chunk import attend_chunk, plan_chunk
from dotcache_amd.page_pool import DevicePagePool, PoolGeometry


def _pools():
    pools = [DevicePagePool(PoolGeometry(64, 32, 16), device="cpu", reserve_bytes=1 << 16, reserve_pages=16) for _ in range(2)]
    for p in pools:
        p.allocate(1, 4, 8, tokens=16)
    return pools


def test_a_workspace_off_16_bytes():
    geo = _lib.geometry(64, 32, 16)
    pool = _lib.Pool(arena=4096, arena_bytes=1 << 20, descs=4096, n_descs=4, geometry=geo)
    rows = _lib.TokenRows(data=4096, token_stride=64, head_stride=64, n_heads=2, dtype=1)
    for off in (1, 4, 8):
        assert _lib.lib().dc_attend_chunk(pool, pool, 4096, 4096, 1, 4096, 1, 0, 0, None, 0, 4, 1, 1, 1, rows, 1.0, rows, 4096 + off,
                                          1 << 20, None) == _lib.DC_EINVAL
    pools = _pools()
    split = plan_chunk(*pools, [1], [6000], kv_heads=1, q_per_kv=1)
    assert split.n_partials > 0
    table = torch.zeros(1, 1, 375, dtype=torch.int32)
    space = torch.zeros(1 << 20, dtype=torch.uint8)
    start = -space.data_ptr() % 16
    for off, match in ((0, "on a GPU"), (1, "16-byte"), (8, "16-byte")):
        with pytest.raises(ValueError, match=match):
            attend_chunk(pools[0], table, pools[1], table, torch.zeros(1, 1, 64), split, workspace=space[start + off:])


def test_a_plan_serves_every_query_type():
    """``dtype`` is checked; the plan does not depend on it."""
    import numpy as np

    plans = [plan_chunk(*_pools(), [5, 90], [700, 300], kv_heads=2, q_per_kv=3, target_items=16, dtype=dt)
             for dt in (None, torch.float32, torch.float16, torch.bfloat16)]
    for p in plans[1:]:
        assert np.array_equal(p.host_items, plans[0].host_items) and np.array_equal(p.host_merges, plans[0].host_merges)
    for dt in (torch.float64, torch.int8, "bf16"):
        with pytest.raises(ValueError, match="dtype"):
            plan_chunk(*_pools(), [5], [700], kv_heads=2, q_per_kv=3, dtype=dt)
