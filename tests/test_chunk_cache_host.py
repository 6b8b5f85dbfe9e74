"""What the caches' chunk calls refuse, before any device work and with the
cache left as it was."""
import numpy as np
import pytest

from dotcache_amd.block_cache import DeviceVllmPagedKVCache
from dotcache_amd.config import DotCacheConfig
from dotcache_amd.kv_cache import DevicePagedKVCache
from dotcache_amd.rotary import RotaryTable

HD, H, HQ = 64, 2, 4


def _paged(batch=1):
    return DevicePagedKVCache(DotCacheConfig(head_dim=HD, group_size=32, tokens_per_page=16), num_hidden_layers=1,
                              num_attention_heads=HQ, num_key_value_heads=H, batch_size=batch, device="cpu")


def _blocks():
    return DeviceVllmPagedKVCache(config=DotCacheConfig(head_dim=HD, group_size=32, tokens_per_page=16), num_hidden_layers=1,
                                  num_attention_heads=HQ, num_key_value_heads=H, block_size=16, device="cpu")


def _table(n=32, hd=HD):
    return RotaryTable(hd, n, device="cpu")


def _step(n, heads, batch=1):
    return np.zeros((batch, heads, n, HD), np.float32)


@pytest.mark.parametrize("call,match", [
    (lambda c: c.append_rotated(0, None, _step(3, H), _step(3, H), 1, None), "expected token_index 0"),
    (lambda c: c.append_rotated(1, None, _step(3, H), _step(3, H), 0, None), "out of range"),
    (lambda c: c.append_rotated(0, None, _step(3, H), _step(2, H), 0, None), "must hold 3 tokens"),
    (lambda c: c.append_rotated(0, _step(2, HQ), _step(3, H), _step(3, H), 0, None), "must hold 3 tokens"),
    (lambda c: c.append_rotated(0, _step(3, H), _step(3, H), _step(3, H), 0, None), "query_step must have shape"),
    (lambda c: c.append_rotated(0, None, _step(3, H), _step(3, H), 0, _table(hd=32)), "another head_dim"),
    (lambda c: c.append_rotated(0, None, _step(3, H), _step(3, H), 0, _table(2)), "positions must lie"),
    (lambda c: c.append_rotated(0, None, _step(3, H), _step(3, H), 0, _table(), positions=[0, 1]), "positions must have shape"),
    (lambda c: c.append_rotated(0, None, _step(3, H), _step(3, H), 0, _table(), positions=[0, -1, 2]), "positions must lie"),
    (lambda c: c.append_rotated(0, None, _step(3, H), _step(3, H), 0, _table(), k_weight=__import__("torch").ones(HD + 1)), "weight must be"),
    (lambda c: c.append_rotated(0, None, _step(3, H), _step(3, H), 0, _table(), k_weight=__import__("torch").ones(HD), eps=-1.0), "eps"),
    (lambda c: c.attend_chunk(0, _step(3, HQ)), "holds 0 tokens"),
    (lambda c: c.attend_chunk(0, _step(3, H)), "query_chunk must have shape"),
])
def test_paged_cache_refusals(call, match):
    c = _paged()
    with pytest.raises(ValueError, match=match):
        call(c)
    assert c.sequence_length(0) == 0 and c.tail_page_id(0, 0, 0) == -1


def test_empty_steps():
    c = _paged(2)
    q = c.append_rotated(0, _step(0, HQ, 2), _step(0, H, 2), _step(0, H, 2), 0, _table())
    assert q.shape == (2, HQ, 0, HD) and c.sequence_length(0) == 0
    assert c.attend_chunk(0, _step(0, HQ, 2)).shape == (2, HQ, 0, HD)
    assert all(x.shape == (2, H, 0, HD) for x in c.read_layer(0))


@pytest.mark.parametrize("call,match", [
    (lambda c: c.write_slots_rotated(0, np.zeros((2, HQ, HD)), np.zeros((3, H, HD)), np.zeros((3, H, HD)), [0, 1, 2], [0, 1, 2], _table()),
     "same number of tokens"),
    (lambda c: c.write_slots_rotated(0, np.zeros((3, H, HD)), np.zeros((3, H, HD)), np.zeros((3, H, HD)), [0, 1, 2], [0, 1, 2], _table()),
     "query_rows must have shape"),
    (lambda c: c.write_slots_rotated(0, None, np.zeros((3, H, HD)), np.zeros((3, H, HD)), [0, 1, 2], [0, 1, 40], _table()),
     "positions must lie"),
    (lambda c: c.write_slots_rotated(0, None, np.zeros((3, H, HD)), np.zeros((3, H, HD)), [0, 1, 2], [0, 1], _table()),
     "one entry per token"),
    (lambda c: c.write_slots_rotated(0, None, np.zeros((3, H, HD)), np.zeros((3, H, HD)), [0, 1], [0, 1, 2], _table()), "one slot per row"),
    (lambda c: c.write_slots_rotated(0, None, np.zeros((3, H, HD)), np.zeros((3, H, HD)), [0, 1, -1], [0, 1, 2], _table()), "non-negative"),
    (lambda c: c.write_slots_rotated(0, None, np.zeros((1, H, HD)), np.zeros((1, H, HD)), [3], [0], _table()), "out of order"),
    (lambda c: c.attend_block_tables(0, np.zeros((1, HQ, HD)), [1], [[0]], [1]), "no pages"),
    (lambda c: c.attend_block_tables(0, np.zeros((1, HQ, HD)), [1], [[0]], [0]), "positive length"),
    (lambda c: c.attend_block_tables(0, np.zeros((1, HQ, HD)), [1, 0], [[0]], [1, 1]), "block_tables must have shape"),
    (lambda c: c.read_block_tables(0, [[0]], [1]), "no pages"),
    (lambda c: c.read_block_tables(0, [[0]], [17]), "more blocks"),
])
def test_block_cache_refusals(call, match):
    c = _blocks()
    with pytest.raises(ValueError, match=match):
        call(c)
    assert not c._fill[0].any() and not c._row_slots[0]


def test_write_slots_rotated_hands_every_row_over_once(monkeypatch):
    """Blocks that fill, whole blocks, a live block and a block reused in the
    call: each row's page, slot, kept row, position and queries."""
    import torch

    c = _blocks()
    seen = []

    def write(self, v_pool, q, k, v, positions, rotary, tables, row, token, *, q_weight, k_weight, eps, out, keep):
        for i in range(k.shape[0]):
            pages = tables[:, int(row[i]), :, 0].tolist()
            kept = None if keep is None or int(keep[2][i]) < 0 else int(keep[2][i])
            seen.append((float(k[i, 0, 0]), int(positions[i]), int(token[i]), pages, kept))
            for x, buf in ((k, keep and keep[0]), (v, keep and keep[1])):
                if kept is not None:
                    for h in range(H):
                        buf[kept + h * keep[3]] = x[i, h]
        out.copy_(q)

    finals = []
    monkeypatch.setattr(type(c.k_pool), "append_rotary_with", write)
    monkeypatch.setattr(type(c.k_pool), "encode_streams_with", lambda self, vp, k, v, t, **kw: finals.append((k.clone(), v.clone())))
    n = 5 + 16 + 11 + 3
    k = torch.arange(n, dtype=torch.float32).view(n, 1, 1).expand(n, H, HD) + 100.0 * torch.arange(H).view(1, H, 1)
    slots = np.concatenate([3 * 16 + np.arange(5), 16 + np.arange(16), 3 * 16 + 5 + np.arange(11), 3 * 16 + np.arange(3)])
    q = torch.randn(n, HQ, HD)
    out = c.write_slots_rotated(0, q, k, -k, slots, np.arange(n) % 32, _table())
    assert torch.equal(out, q)
    assert [s[0] for s in seen] == list(range(n)) and [s[1] for s in seen] == [i % 32 for i in range(n)]
    assert [s[2] for s in seen] == (slots % 16).tolist()
    whole = seen[5:21]
    assert all(s[4] is None and min(min(p) for p in s[3]) >= 0 for s in whole)  # straight into final pages
    assert all(s[4] is not None and s[3] == [[-1] * H] * 2 for s in seen[21:32])  # they fill the block: kept alone
    assert all(s[4] is not None and min(min(p) for p in s[3]) >= 0 for s in seen[32:])
    assert len(finals) == 1
    order = torch.tensor([*range(5), *range(21, 32)], dtype=torch.float32)
    for h in range(H):
        assert torch.equal(finals[0][0][h, :, 0], order + 100 * h) and torch.equal(finals[0][1][h, :, 0], -(order + 100 * h))
    assert c._fill[0][3] == 3 and c._fill[0][1] == 16
