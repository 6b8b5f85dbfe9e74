"""Chunk attention with masks, capped and distance-lowered scores against fp64
numpy on the pages' own values: windows with and without sinks, prefixes,
documents, ranges of any kind with rows that attend nothing, at every kernel
(16-bit and fp32 queries, few and many rows, whole and odd geometries), with
ranges cut and joined, values that are not finite where no row looks, pages
that no row needs, graphs and streams."""
import numpy as np
import pytest

from dotcache_amd.chunk import ChunkMask
from tests.test_chunk_mask_host import seen_by_ranges, sees
from tests.test_gpu_chunk import _Batch, _dt

pytestmark = pytest.mark.gpu


def slopes_of(Hq):
    return (2.0 ** (-8.0 * (np.arange(Hq) + 1) / Hq)).astype(np.float32)


def want_rule(batch, q, new, n_q, scale, dtype, seen, cap=None, slopes=None):
    """fp64 outputs [tokens, Hq, hd] and a bound on a kernel's error.

    A logit is off by delta: 16-bit queries have operands rounded to fp16, 2^-11
    each, so 2^-10 sum |q| |k| (fp32: hd + 4 products and sums of 2^-24); the cap's
    slope is at most 1 and its own arithmetic (an exponential, a sum, a reciprocal and
    a product of values below 2) loses 2^-20 cap; a product with the distance,
    and the sum, 2^-22 of each term.  So a weight is off by e^delta and the
    weights' sum by the mean D of that: sum p |v| (e^2delta - 1 + D).  A weight and a value are rounded to
    fp16 once more (2^-11 each; fp32: the sums over tokens, 2^-24 each), weights
    below the fp16 range lose 2^-25 of the largest, and the output's own rounding comes last."""
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    half = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
    per = (batch.hd + 4) * 2.0 ** -24 if dtype == "f32" else 2.0 ** -10
    t0 = 0
    for b, n in enumerate(new):
        c = batch.ctx[b]
        ok = seen(b, t0, n)
        away = np.abs(np.arange(c - n, c)[:, None] - np.arange(c)[None, :])
        for h in range(batch.H if n else 0):
            k, v = (x[b, h, :c] for x in batch.rows)
            k, v = np.where(ok.any(0)[:, None], k, 0.0), np.where(ok.any(0)[:, None], v, 0.0)  # (others may hold anything)
            for j in range(h * n_q, (h + 1) * n_q):
                x = q[t0: t0 + n, j]
                s = scale * (x @ k.T)
                delta = per * abs(scale) * (np.abs(x) @ np.abs(k).T) + 2.0 ** -20
                if cap:
                    s = cap * np.tanh(s / cap)
                    delta = delta + cap * 2.0 ** -20
                if slopes is not None:
                    s = s - float(slopes[j]) * away
                    delta = delta + 2.0 ** -22 * (abs(float(slopes[j])) * away + np.abs(s))
                s = np.where(ok, s, -np.inf)
                top = s.max(axis=1, keepdims=True)
                p = np.exp(s - np.where(np.isfinite(top), top, 0.0))
                p /= np.maximum(p.sum(axis=1, keepdims=True), 1e-300)
                out[t0: t0 + n, j] = p @ v
                e = np.expm1(2 * np.where(ok, delta, 0.0))
                size = p @ np.abs(v)
                own = c * 2.0 ** -24 + 2.0 ** -21 if dtype == "f32" else 2.0 ** -10 * (1 + 2.0 ** -6)
                low = 0.0 if dtype == "f32" else c * 2.0 ** -25 * np.abs(v).max(initial=0.0)
                bound[t0: t0 + n, j] = (p * e) @ np.abs(v) + ((p * e).sum(1, keepdims=True) + own) * size + low * ok.any(1)[:, None] \
                    + half * np.abs(out[t0: t0 + n, j]) + 2.0 ** -20
        t0 += n
    return out, bound


def check_rule(batch, new, n_q, dtype, rng, mask=None, cap=None, slopes=False, scale=None, plan=None, q=None, size=0.5, **kw):
    import torch

    T, Hq, hd = int(sum(new)), batch.H * n_q, batch.hd
    if q is None:
        q = torch.from_numpy((rng.normal(size=(T, Hq, hd)) * size).astype(np.float32)).to(_dt(dtype)).cuda()
    scale = 1.0 / np.sqrt(hd) if scale is None else scale
    sl = slopes_of(Hq) * (1.0 if slopes is True else slopes) if slopes is not False else None
    plan = plan or batch.plan(new, n_q, dtype=q.dtype, mask=mask)
    got = batch.attend(q, plan, scale, cap=cap, slopes=None if sl is None else torch.from_numpy(sl).cuda(), **kw)
    assert got.shape == q.shape and got.dtype == q.dtype

    def seen(b, t0, n):
        c = batch.ctx[b]
        if isinstance(mask, np.ndarray):
            return seen_by_ranges(mask[t0: t0 + n], c)
        return sees(mask or ChunkMask(), b, c)[c - n:]

    want, bound = want_rule(batch, q[:T].double().cpu().numpy(), new, n_q, scale, dtype, seen, cap, sl)
    err = np.abs(got[:T].double().cpu().numpy() - want)
    assert np.all(err <= bound), float(np.max(err / bound))
    return q, got, plan


RULES = {"cap": dict(cap=4.0), "distance": dict(slopes=True), "window": dict(mask=ChunkMask(window=50)),
         "sinks": dict(mask=ChunkMask(window=70, sinks=5)), "prefix": dict(mask=ChunkMask(prefix=(100, 0, 7))),
         "documents": dict(mask=ChunkMask(documents=[[0, 3, 290, 300, 301], [], [0, 5]])),
         "all": dict(mask=ChunkMask(window=60, sinks=3, prefix=(120, 1, 9), documents=[[0, 130, 250], [0, 20], []]), cap=3.0, slopes=True)}


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 96, 256])
@pytest.mark.parametrize("rule", list(RULES))
def test_rules(rule, hd, dtype):
    """Row tiles, drafted tokens and a decode of three sequences in one call."""
    rng = np.random.default_rng(hd + len(rule))
    print(f"chunk rule {rule} {hd} {dtype}", flush=True)
    batch = _Batch(rng, [331, 200, 9], 2, hd, 32, "a4", "s4")
    check_rule(batch, [140, 3, 1], 3, dtype, rng, validate=True, **RULES[rule])


@pytest.mark.parametrize("rule", ["sinks", "all"])
@pytest.mark.parametrize("key,value,hd,gs,P", [("a8", "a3", 128, (32, 32), 48), ("m3", "s8", 80, (16, 32), 16), ("s2", "m3_i8", 30, (32, 32), 20),
                                               ("m3", "m3", 128, (32, 32), 24), ("s8", "m3", 64, (32, 64), 128), ("m3", "a4", 256, (32, 32), 8),
                                               ("a4", "a4", 1, (32, 32), 16)])
def test_formats_and_geometries(key, value, hd, gs, P, rule):
    rng = np.random.default_rng(hd + P)
    batch = _Batch(rng, [331, 200, 9], 1, hd, P, key, value, gs)
    for dtype in ("f32", "bf16"):
        print(f"chunk rule {rule} {key} {value} {hd} {P} {dtype}", flush=True)
        check_rule(batch, [97, 5, 1], 5, dtype, rng, **RULES[rule])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new", [[1, 1], [9, 2], [300, 40]])
def test_cut_ranges_and_gaps(new, dtype):
    """Long contexts cut into many parts, with items on both sides of a gap, and whole."""
    rng = np.random.default_rng(sum(new))
    batch = _Batch(rng, [1900, 1500], 2, 64, 64, "a4", "s4")
    for mask in (ChunkMask(window=700, sinks=200), ChunkMask(window=129, sinks=4), ChunkMask(window=4000), None):
        for target in (1, 40, 512):
            print(f"chunk rule cut {new} {dtype} {mask} {target}", flush=True)
            plan = batch.plan(new, 4, mask=mask, target_items=target)
            check_rule(batch, new, 4, dtype, rng, mask=mask, cap=5.0, slopes=True, plan=plan)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_any_ranges_and_rows_that_attend_nothing(dtype):
    rng = np.random.default_rng(5)
    batch = _Batch(rng, [700, 30, 250], 2, 128, 64, "a4", "a4")
    new = [150, 30, 1]
    for last in (0, 1):  # the decode attends nothing, or one token
        r = np.zeros((181, 4), dtype=np.int64)
        t = 0
        for n, c in zip(new, batch.ctx):
            a = np.sort(rng.integers(0, c + 1, size=(n, 4)), axis=1)
            r[t: t + n] = np.where(rng.random((n, 1)) < 0.5, a, a[:, [2, 3, 0, 1]])
            t += n
        r[40:100:3] = 0
        r[100:170] = [5, 5, 9, 9]
        r[-1] = [7, 7, 249, 249 + last]
        print(f"chunk ranges {dtype} {last}", flush=True)
        _, got, _ = check_rule(batch, new, 3, dtype, rng, mask=r, slopes=True, validate=True)
        assert not got[40:100:3].any() and not got[100:170].any() and bool(got[-1].any()) == bool(last)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_values_that_are_not_finite_stay_with_rows_that_see_them(hd, dtype):
    """Infinities and NaN in keys and values outside every row's window change
    nothing; inside some rows' ranges they reach those rows and no other."""
    import torch

    rng = np.random.default_rng(hd)
    batch = _Batch(rng, [400], 1, hd, 32, "m3", "m3", tail=False)
    mask = ChunkMask(window=64)
    print(f"chunk rule not finite {hd} {dtype}", flush=True)
    q, clean, plan = check_rule(batch, [100], 2, dtype, rng, mask=mask)
    bad = torch.full((1, hd), float("nan"), device="cuda")
    bad[0, ::2] = float("inf")
    for side in (0, 1):
        for u in (0, 200, 236):  # (row 0 is token 300 and attends 237 on)
            batch.pools[side].encode_rows(bad, [batch.host[side][0, 0, u // 32]], [u % 32])
    again = batch.attend(q, plan, 1.0 / np.sqrt(hd))
    assert torch.equal(clean, again)
    u = 350  # rows of tokens 350 .. 399 see it
    batch.pools[1].encode_rows(bad, [batch.host[1][0, 0, u // 32]], [u % 32])
    some = batch.attend(q, plan, 1.0 / np.sqrt(hd))
    assert torch.equal(some[:50], clean[:50]) and not torch.isfinite(some[50:]).any()


def test_pages_out_of_sight_need_not_exist():
    import torch

    rng = np.random.default_rng(9)
    batch = _Batch(rng, [900, 640], 2, 64, 32, "a4", "s4")
    mask = ChunkMask(window=100, sinks=4)
    for new in ([1, 1], [90, 33]):
        for dtype in ("f32", "f16"):
            print(f"chunk rule pages {new} {dtype}", flush=True)
            q, whole, plan = check_rule(batch, new, 2, dtype, rng, mask=mask)
            kept = [t.clone() for t in batch.tables]
            for t in batch.tables:
                t[0, :, 1:(900 - new[0] - 99) // 32] = -1
                t[1, :, 1:(640 - new[1] - 99) // 32] = 10 ** 6
            assert torch.equal(batch.attend(q, plan, 0.125, validate=True), whole)
            batch.tables = kept
    with pytest.raises((ValueError, IndexError, KeyError)):
        batch.tables[0][0, :, 28] = 10 ** 6
        batch.attend(q, plan, 0.125, validate=True)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
def test_scales_caps_and_slopes_of_either_sign(scale):
    """Scores far past the cap, and slopes that favour far tokens."""
    rng = np.random.default_rng(3)
    batch = _Batch(rng, [500, 70], 2, 64, 64, "a4", "s4")
    for dtype in ("f32", "f16"):
        for new in ([120, 2], [1, 1]):
            print(f"chunk rule scale {scale} {dtype} {new}", flush=True)
            check_rule(batch, new, 2, dtype, rng, cap=1.5, scale=scale)
            check_rule(batch, new, 2, dtype, rng, slopes=-1.0, cap=2.0, scale=scale, mask=ChunkMask(window=200))


def test_large_products_stay_at_the_cap():
    """Products past any float's exponent give the cap, not a NaN."""
    import torch

    rng = np.random.default_rng(8)
    batch = _Batch(rng, [200], 1, 64, 32, "m3", "m3")
    for dtype in ("f32", "f16"):
        q = torch.full((1, 1, 64), 30000.0, device="cuda", dtype=_dt(dtype))
        q[..., ::2] *= -1
        got = batch.attend(q, batch.plan([1], 1), 1e30, cap=2.0)
        k, v = (x[0, 0] for x in batch.rows)
        p = np.exp(2.0 * np.sign(k[:200] @ q.double().cpu().numpy()[0, 0]))
        assert np.max(np.abs(got.double().cpu().numpy()[0, 0] - (p / p.sum()) @ v[:200])) < 2e-3


def test_strides_padding_and_far_tokens():
    """Queries and outputs that are views, rows behind the plan's, and the last
    tokens of a long context lowered by their distance."""
    import torch

    rng = np.random.default_rng(4)
    batch = _Batch(rng, [20000, 300], 1, 64, 64, "a4", "s4")
    mask = ChunkMask(window=30, sinks=64)
    plan = batch.plan([3, 40], 2, mask=mask)
    wide = torch.from_numpy(rng.normal(size=(50, 5, 80)).astype(np.float32) * 0.5).half().cuda()
    out = torch.full((50, 3, 64), 7.0, dtype=torch.float16, device="cuda")
    _, got, _ = check_rule(batch, [3, 40], 2, "f16", rng, mask=mask, slopes=True, cap=6.0, plan=plan, q=wide[:, 1:3, 5:69], out=out[:, 1:])
    assert got.data_ptr() == out[:, 1:].data_ptr() and bool((out[43:] == 7).all()) and bool((out[:, 0] == 7).all())
    check_rule(batch, [3, 40], 2, "f32", rng, slopes=0.01, mask=mask)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_distances_of_far_tokens(dtype):
    """Past token 2^24 the distance still counts whole tokens: the last ones of
    a context whose other pages are not there weigh as in a short one."""
    import torch

    from dotcache_amd.chunk import attend_chunk, plan_chunk

    rng = np.random.default_rng(1)
    far, P = 2 ** 24 + 3 * 64, 64
    batch = _Batch(rng, [64], 1, 64, P, "a4", "a4", tail=False)
    q = torch.from_numpy(rng.normal(size=(3, 2, 64)).astype(np.float32)).to(_dt(dtype)).cuda()
    sl = torch.tensor([0.9, 0.3], device="cuda")
    mask = ChunkMask(window=40)
    near = batch.attend(q, batch.plan([3], 2, mask=mask), 0.125, slopes=sl)
    tables = [torch.full((1, 1, (far + 64) // P), -1, dtype=torch.int32, device="cuda") for _ in range(2)]
    for t, kept in zip(tables, batch.tables):
        t[0, 0, -1] = kept[0, 0, 0]
    plan = plan_chunk(*batch.pools, [3], [far + 64], kv_heads=1, q_per_kv=2, mask=mask)
    got = attend_chunk(batch.pools[0], tables[0], batch.pools[1], tables[1], q, plan, query_scale=0.125, slopes=sl)
    # (the same pages, tokens and distances; the wavefronts may take them in another order)
    assert float((got.double() - near.double()).abs().max()) <= 4 * torch.finfo(q.dtype).eps * float(near.abs().max())


def test_replays_and_streams():
    """A captured call replayed with other queries and slopes, eager work in
    between, and the same call on another stream."""
    import torch

    rng = np.random.default_rng(6)
    batch = _Batch(rng, [1200, 300], 2, 128, 64, "a4", "s4")
    new, mask = [1, 70], ChunkMask(window=500, sinks=4)
    plan = batch.plan(new, 2, mask=mask)
    qs = [torch.from_numpy(rng.normal(size=(71, 4, 128)).astype(np.float32)).bfloat16().cuda() for _ in range(3)]
    sl = [torch.from_numpy(slopes_of(4) * f).cuda() for f in (1.0, 0.3, 0.1)]
    want = [batch.attend(q, plan, 0.1, cap=4.0, slopes=s) for q, s in zip(qs, sl)]
    q, s, out = qs[0].clone(), sl[0].clone(), torch.empty_like(qs[0])
    from dotcache_amd.chunk import workspace_bytes

    work = torch.empty(workspace_bytes(plan, 128), dtype=torch.uint8, device="cuda")
    call = lambda: batch.attend(q, plan, 0.1, cap=4.0, slopes=s, out=out, workspace=work)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(out, want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in (1, 2, 0, 1):
        q.copy_(qs[i])
        s.copy_(sl[i])
        graph.replay()
        assert torch.equal(out, want[i])
        out.zero_()
        torch.cuda.synchronize()


def test_caches_take_masks_and_scores():
    """Both caches: layers of one step with different masks, heads in any
    order, against the call on their pages."""
    import torch

    from dotcache_amd.config import DotCacheConfig
    from dotcache_amd.kv_cache import DevicePagedKVCache

    rng = np.random.default_rng(2)
    cfg = DotCacheConfig(head_dim=64, group_size=32, bits_k=4, bits_v=4, tokens_per_page=32)
    cache = DevicePagedKVCache(cfg, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, batch_size=2)
    x = [torch.from_numpy(rng.normal(size=(2, 2, 150, 64)).astype(np.float32)).cuda() for _ in range(4)]
    for layer in range(2):
        cache.ingest_prefill_cache(layer, x[2 * layer], x[2 * layer + 1])
    q = torch.from_numpy(rng.normal(size=(2, 4, 20, 64)).astype(np.float32)).cuda()
    sl = torch.from_numpy(slopes_of(4)).cuda()
    order = [1, 0, 1, 0]  # query heads 1 and 3 read KV head 0
    for layer, mask in ((0, ChunkMask(window=33, sinks=2)), (1, None), (0, ChunkMask(documents=[[0, 140], [0]])), (1, None)):
        got = cache.attend_chunk(layer, q, order, query_scale=0.125, mask=mask, cap=5.0, slopes=sl).double().cpu().numpy()
        k, v = (y.double().cpu().numpy() for y in cache.read_layer(layer))
        for b in range(2):
            ok = sees(mask or ChunkMask(), b, 150)[130:]
            for j in range(4):
                s = 5.0 * np.tanh(0.125 * (q[b, j].double().cpu().numpy() @ k[b, order[j]].T) / 5.0)
                s = s - float(sl[j]) * np.abs(np.arange(130, 150)[:, None] - np.arange(150))
                p = np.exp(np.where(ok, s, -np.inf))
                p /= p.sum(1, keepdims=True)
                # (fp32 throughout: 150 tokens and 64 channels, values below 8)
                assert np.max(np.abs(got[b, j] - p @ v[b, order[j]])) < 1e-4
    assert len(cache._chunk_plan[1]) == 3
    with pytest.raises(ValueError):
        cache.attend_chunk(0, q, query_scale=0.125, mask=np.zeros((40, 4), dtype=np.int32))


@pytest.mark.parametrize("layout", ["group_major", "token_major"])
@pytest.mark.parametrize("hd,n_q,new", [(64, 3, 5), (64, 7, 9), (128, 7, 1), (128, 4, 6), (128, 7, 6), (256, 4, 1), (256, 5, 3)])
def test_few_rows_of_4_bit_pages(hd, n_q, new, layout):
    """Pools of 4-bit pages alone take kernels of their own; once a pool has
    held an 8-bit page, the same call takes the others: the same outputs, plain and
    with a rule, tails of fp16 among the pages."""
    import torch

    rng = np.random.default_rng(hd + n_q)
    for key, value, tail in (("a4", "s4", True), ("s4", "a4", False), ("a4", "a4", True)):
        print(f"few rows of 4 bits {hd} {n_q} {new} {layout} {key} {value}", flush=True)
        batch = _Batch(rng, [700, 65, 32], 2, hd, 32, key, value, layout=layout, tail=tail)
        n = [new, min(new, 3), 1]
        calls = [dict(mask=ChunkMask(window=200, sinks=3), cap=5.0, slopes=True), dict()]
        first = [check_rule(batch, n, n_q, "bf16", rng, **kw) for kw in calls]
        for p in batch.pools:
            p.allocate(1, 8, 1)
        for kw, (q, got, plan) in zip(calls, first):
            sl = torch.from_numpy(slopes_of(2 * n_q)).cuda() if kw.get("slopes") else None
            assert torch.equal(batch.attend(q, plan, 1.0 / np.sqrt(hd), cap=kw.get("cap"), slopes=sl), got)


def test_block_cache_takes_masks_and_scores():
    """A serving engine's mixed batch: window and cap over block tables, against
    the same cache's dense rows."""
    import torch

    from dotcache_amd.block_cache import DeviceVllmPagedKVCache
    from dotcache_amd.config import DotCacheConfig

    rng = np.random.default_rng(7)
    cfg = DotCacheConfig(head_dim=64, group_size=32, bits_k=4, bits_v=4, tokens_per_page=16)
    cache = DeviceVllmPagedKVCache(config=cfg, num_hidden_layers=1, num_attention_heads=4, num_key_value_heads=2, block_size=16)
    lens, new = [70, 33], [20, 1]
    tables = [[7, 2, 9, 4, 0], [5, 1, 3]]
    for b, n in enumerate(lens):
        x = [torch.from_numpy(rng.normal(size=(n, 2, 64)).astype(np.float32)).cuda() for _ in range(2)]
        cache.write_slots(0, *x, [16 * tables[b][t // 16] + t % 16 for t in range(n)])
    q = torch.from_numpy(rng.normal(size=(21, 4, 64)).astype(np.float32)).cuda()
    padded = [t + [0] * (5 - len(t)) for t in tables]
    mask = ChunkMask(window=18, sinks=2, prefix=(60, 0))
    sl = torch.from_numpy(slopes_of(4)).cuda()
    got = cache.attend_block_tables(0, q, new, padded, lens, query_scale=0.125, mask=mask, cap=3.0, slopes=sl).double().cpu().numpy()
    k, v = (y.double().cpu().numpy() for y in cache.read_block_tables(0, padded, lens))
    t0 = u0 = 0
    for b, (n, c) in enumerate(zip(new, lens)):
        ok = sees(mask, b, c)[c - n:]
        for j in range(4):
            kk, vv = (y[u0: u0 + c, j // 2] for y in (k, v))
            s = 3.0 * np.tanh(0.125 * (q[t0: t0 + n, j].double().cpu().numpy() @ kk.T) / 3.0)
            s = s - float(sl[j]) * np.abs(np.arange(c - n, c)[:, None] - np.arange(c))
            p = np.exp(np.where(ok, s, -np.inf))
            # (fp32 throughout, values below 8)
            assert np.max(np.abs(got[t0: t0 + n, j] - p / p.sum(1, keepdims=True) @ vv)) < 1e-4
        t0, u0 = t0 + n, u0 + c
