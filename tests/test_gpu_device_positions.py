"""Positions that live on the device and lie outside the rotation's table: the
caches refuse them before anything is counted, as they do positions on the
host."""
import numpy as np
import pytest

from dotcache_amd.config import DotCacheConfig

pytestmark = pytest.mark.gpu

HD, H, HQ, P = 64, 2, 4, 16


def _cfg():
    return DotCacheConfig(head_dim=HD, group_size=32, tokens_per_page=P, bits_k=4, bits_v=4)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("batch", [1, 2])
def test_paged_cache(batch, wide):
    """On a tail page that has held other tokens, one short of full and just
    begun: the refused call changes nothing, the next one goes on."""
    import torch

    from dotcache_amd.kv_cache import DevicePagedKVCache
    from dotcache_amd.rotary import RotaryTable

    make = lambda: DevicePagedKVCache(_cfg(), num_hidden_layers=1, num_attention_heads=HQ, num_key_value_heads=H, batch_size=batch)  # noqa: E731
    cache, plain = make(), make()
    rotary = RotaryTable(HD, 64)
    dt = torch.int64 if wide else torch.int32
    torch.manual_seed(batch)
    at = 0
    for n, bad in ((P - 1, 64), (1, -1), (3, 2 ** 31 - 1), (P, 64)):
        x = [torch.randn(batch, h, n, HD, device="cuda") for h in (HQ, H, H)]
        pos = torch.arange(at, at + n, device="cuda", dtype=dt)
        for shape in ((n,), (batch, n)):
            wrong = pos.expand(shape).clone()
            wrong[(*[-1] * (len(shape) - 1), n // 2)] = bad
            with pytest.raises(ValueError, match="positions must lie"):
                cache.append_rotated(0, *x, at, rotary, positions=wrong)
            assert cache.sequence_length(0) == at
        q = cache.append_rotated(0, *x, at, rotary, positions=pos)
        assert torch.equal(q, plain.append_rotated(0, *x, at, rotary))
        at += n
        for a, b in zip(cache.read_layer(0), plain.read_layer(0)):
            assert torch.equal(a, b)


def test_block_cache():
    import torch

    from dotcache_amd.block_cache import DeviceVllmPagedKVCache
    from dotcache_amd.rotary import RotaryTable

    cache = DeviceVllmPagedKVCache(config=_cfg(), num_hidden_layers=1, num_attention_heads=HQ, num_key_value_heads=H, block_size=P)
    rotary = RotaryTable(HD, 64)
    x = [torch.randn(5, h, HD, device="cuda") for h in (HQ, H, H)]
    slots = 2 * P + np.arange(5)
    pos = torch.arange(5, device="cuda")
    for bad in (64, -1, 2 ** 40):
        wrong = pos.clone()
        wrong[3] = bad
        with pytest.raises(ValueError, match="positions must lie"):
            cache.write_slots_rotated(0, *x, slots, wrong, rotary)
        with pytest.raises(ValueError, match="no pages"):
            cache.read_block_tables(0, [[2]], [5])
    cache.write_slots_rotated(0, *x, slots, pos, rotary)
    k, v = cache.read_block_tables(0, [[2]], [5])
    assert torch.isfinite(k).all() and torch.equal(v, x[2].half().float())
