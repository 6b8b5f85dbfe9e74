"""Sequences whose blocks before the last are not full: the calls that place
tokens by their position refuse them, before any device work."""
import numpy as np
import pytest

from dotcache_amd.block_cache import DeviceVllmPagedKVCache
from dotcache_amd.config import DotCacheConfig

HD, H, HQ, P = 64, 2, 4, 16


@pytest.fixture
def cache(monkeypatch):
    """Block 1 with 10 tokens, block 2 full, block 3 with 6."""
    c = DeviceVllmPagedKVCache(config=DotCacheConfig(head_dim=HD, group_size=32, tokens_per_page=P), num_hidden_layers=1,
                               num_attention_heads=HQ, num_key_value_heads=H, block_size=P, device="cpu")
    monkeypatch.setattr(type(c.k_pool), "encode_rows_with", lambda self, *a, **kw: None)
    slots = np.concatenate([P + np.arange(10), 2 * P + np.arange(16), 3 * P + np.arange(6)])
    c.write_slots(0, np.zeros((32, H, HD)), np.zeros((32, H, HD)), slots)
    return c


@pytest.mark.parametrize("tables,lens", [([[1, 2]], [26]), ([[2, 3], [1, 2]], [22, 26])])
def test_a_short_block_before_the_last(cache, tables, lens):
    new = [0] * (len(lens) - 1) + [2]
    with pytest.raises(ValueError, match="before its last"):
        cache.attend_block_tables(0, np.zeros((2, HQ, HD)), new, tables, lens)
    with pytest.raises(ValueError, match="before its last"):
        cache.read_block_tables(0, tables, lens)


def test_full_blocks_pass(cache):
    """(as far as the launch, which needs a GPU)"""
    for call in (lambda: cache.attend_block_tables(0, np.zeros((2, HQ, HD)), [2], [[2, 1]], [26]),
                 lambda: cache.read_block_tables(0, [[2, 3], [1, 0]], [22, 10])):
        with pytest.raises(ValueError, match="on a GPU"):
            call()
