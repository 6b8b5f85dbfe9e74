"""A cache's chunk attention on two streams at once and under capture."""
import numpy as np
import pytest

from dotcache_amd.config import DotCacheConfig

pytestmark = pytest.mark.gpu

HD, H, HQ, P = 64, 2, 4, 64


def _cache(tokens):
    import torch

    from dotcache_amd.kv_cache import DevicePagedKVCache

    cache = DevicePagedKVCache(DotCacheConfig(head_dim=HD, group_size=32, tokens_per_page=P), num_hidden_layers=2,
                               num_attention_heads=HQ, num_key_value_heads=H)
    torch.manual_seed(tokens)
    for lid in range(2):
        cache.ingest_prefill_cache(lid, *torch.randn(2, 1, H, tokens, HD, device="cuda"))
    return cache


def test_two_streams():
    """Layers of one cache attended side by side, with chunks of two lengths in
    turn, all of them cut: no call takes another's plan or partial results."""
    import torch

    cache = _cache(5000)
    q = {n: torch.randn(1, HQ, n, HD, device="cuda").half() for n in (3, 9, 70)}
    want = {(lid, n): cache.attend_chunk(lid, x, query_scale=0.125) for lid in range(2) for n, x in q.items()}
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(12):
        for lid, st in enumerate(streams):
            n = (3, 9, 70)[(i + lid) % 3]
            with torch.cuda.stream(st):
                got.append((lid, n, cache.attend_chunk(lid, q[n], query_scale=0.125)))
    torch.cuda.synchronize()
    for lid, n, y in got:
        assert torch.equal(y, want[lid, n])


@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
def test_capture_is_refused():
    """A captured call would go on reading a plan that the cache drops with its
    next lengths; the cache goes on as before."""
    import torch

    cache = _cache(300)
    q = torch.randn(1, HQ, 5, HD, device="cuda").half()
    want = cache.attend_chunk(0, q)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(graph):
            cache.attend_chunk(0, q)
    torch.cuda.synchronize()
    assert torch.equal(cache.attend_chunk(0, q), want)


def test_what_a_call_keeps(monkeypatch):
    """One plan for a step's layers on a stream, none across streams; partial
    results in memory of the call's own."""
    import torch

    from dotcache_amd import chunk

    cache = _cache(700)
    seen = []
    real = chunk.attend_chunk
    monkeypatch.setattr(chunk, "attend_chunk", lambda *a, **kw: (seen.append((a[5], kw.get("workspace"))), real(*a, **kw))[1])
    q = torch.randn(1, HQ, 5, HD, device="cuda").half()
    side = torch.cuda.Stream()
    for st in (torch.cuda.current_stream(), side):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            for lid in range(2):
                cache.attend_chunk(lid, q)
    torch.cuda.synchronize()
    plans = [p for p, _ in seen]
    assert plans[0] is plans[1] and plans[2] is plans[3] and plans[0] is not plans[2]
    assert all(w is None for _, w in seen)
