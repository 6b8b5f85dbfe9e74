"""The pool's append leaves a token whose position lies outside the rotation's
table out of the pages and of the kept fp32 rows alike."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

H, P = 2, 16


@pytest.mark.parametrize("hd", [64, 30])
def test_kept_rows_follow_the_pages(hd):
    import torch

    from dotcache_amd.page_pool import DevicePagePool, PoolGeometry
    from dotcache_amd.rotary import RotaryTable

    pools = [DevicePagePool(PoolGeometry(hd, 32, P), reserve_bytes=1 << 16, reserve_pages=16) for _ in range(2)]
    tables = torch.from_numpy(np.stack([p.allocate(0, 0, H, tokens=P).reshape(1, H, 1) for p in pools]).astype(np.int32)).cuda()
    rotary = RotaryTable(hd, 10)
    x = torch.randn(4, 2 * H, hd, device="cuda")
    pos = torch.tensor([3, 10, -1, 9], device="cuda", dtype=torch.int32)
    keep = torch.full((2, H * P, hd), 7.0, device="cuda")
    pools[0].append_rotary_with(pools[1], None, x[:, :H], x[:, H:], pos, rotary, tables, np.zeros(4, np.int32), np.arange(4),
                                keep=(keep[0], keep[1], np.arange(4), P))
    got = pools[0].read_tokens_with(pools[1], tables, np.zeros(4, np.int32), np.arange(4))
    kept = keep.view(2, H, P, hd)[:, :, :4].transpose(1, 2)
    for t, in_table in enumerate((True, False, False, True)):
        for i in range(2):
            if in_table:
                assert torch.equal(kept[i, t].half().float(), got[i][t])
            else:
                assert torch.all(kept[i, t] == 7.0) and torch.all(got[i][t] == 0)
    assert torch.all(keep.view(2, H, P, hd)[:, :, 4:] == 7.0)
