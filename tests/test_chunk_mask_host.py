"""Masks of the chunk attention, their plans and refusals, on the CPU."""
import numpy as np
import pytest
import torch

from dotcache_amd import _lib
from dotcache_amd.chunk import ChunkMask, attend_chunk, plan_chunk
from tests.test_chunk_host import _plan, _pools


def sees(mask, b, ctx):
    """[ctx, ctx] truth values by the mask's definition: row i attends column u."""
    i, u = np.arange(ctx)[:, None], np.arange(ctx)[None, :]
    prefix = 0 if mask.prefix is None else mask.prefix[b] if isinstance(mask.prefix, tuple) else mask.prefix
    starts = np.asarray((mask.documents[b] if mask.documents is not None else ()) or (0,))
    doc = np.searchsorted(starts, np.arange(ctx), side="right") - 1
    ok = (doc[i] == doc[u]) & ((u <= i) | (u < prefix))
    if mask.window is not None:
        ok &= (u > i - mask.window) | (u - starts[doc][u] < mask.sinks)
    return ok


def seen_by_ranges(ranges, ctx):
    u = np.arange(ctx)[None, :]
    r = ranges[:, :, None]
    return ((u >= r[:, 0]) & (u < r[:, 1])) | ((u >= r[:, 2]) & (u < r[:, 3]))


MASKS = [dict(window=1), dict(window=7, sinks=3), dict(window=40), dict(window=300, sinks=1), dict(prefix=1), dict(prefix=(90, 0, 25)),
         dict(prefix=20, window=6, sinks=2), dict(documents=[[0, 5, 60], [0], [0, 24]]), dict(documents=((0, 1, 2, 3), (), (0,)), window=9, sinks=4),
         dict(documents=[[0, 30], [], [0, 10]], prefix=(50, 1, 25))]


@pytest.mark.parametrize("kw", MASKS)
def test_ranges_are_the_mask(kw):
    mask = ChunkMask(**kw)
    new, ctx = [90, 1, 13], [90, 61, 25]
    r = mask.ranges(new, ctx)
    assert r.dtype == np.int32 and r.shape == (sum(new), 4) and np.all(r[:, 0] <= r[:, 1]) and np.all(r[:, 2] <= r[:, 3])
    t = 0
    for b, (n, c) in enumerate(zip(new, ctx)):
        assert np.array_equal(seen_by_ranges(r[t: t + n], c), sees(mask, b, c)[c - n:])
        t += n
    assert mask == ChunkMask(**kw) and hash(mask) == hash(ChunkMask(**kw))


@pytest.mark.parametrize("target", [1, 64, 512])
@pytest.mark.parametrize("kw", [dict(window=100), dict(window=100, sinks=4), dict(window=129, sinks=300), dict(prefix=(700, 0, 30, 0, 2000)),
                                dict(documents=[list(range(0, 900, 37)), [], [0, 20], [0], [0, 2500]], window=2000, sinks=2)])
def test_items_cover_what_rows_attend(kw, target):
    H, n_q, new, ctx = 2, 3, [700, 1, 43, 1, 200], [900, 5000, 43, 4, 3300]
    plan = _plan(new, ctx, H, n_q, target_items=target, mask=ChunkMask(**kw))
    start = np.concatenate([[0], np.cumsum(new)])
    assert plan.host_gaps.shape == (plan.n_items, 2) and plan.ranges.shape == (sum(new), 4)
    tiles = {}
    for x, gap in zip(plan.host_items.tolist(), plan.host_gaps.tolist()):
        x = dict(zip(_lib.CHUNK_ITEM_FIELDS, x))
        if x["seq"] < 0:
            continue
        assert x["kv_begin"] % (32 if gap == [-1, -1] else 128) == 0 and x["kv_begin"] < x["kv_end"] <= ctx[x["seq"]]
        taken = np.zeros(ctx[x["seq"]], dtype=int)
        taken[x["kv_begin"]: x["kv_end"]] = 1
        if gap != [-1, -1]:
            assert gap[0] % 128 == 0 and gap[1] % 128 == 0 and x["kv_begin"] < gap[0] < gap[1] < x["kv_end"]
            taken[gap[0]: gap[1]] = 0
        tiles.setdefault((x["seq"], x["kv_head"], x["row_begin"], x["row_end"]), []).append(taken)
    assert len(tiles) == sum(-(-n * n_q // 256) for n in new) * H
    for (b, h, r0, r1), parts in tiles.items():
        taken = np.sum(parts, axis=0)
        rows = plan.host_ranges[start[b] + r0 // n_q: start[b] + (r1 - 1) // n_q + 1]
        want = seen_by_ranges(rows, ctx[b]).any(axis=0)
        assert taken.max() == 1 and np.all(taken[want] == 1)
        # nothing beyond the ranges' ends in steps of 128
        steps = np.add.reduceat(want, np.arange(0, ctx[b], 128)) > 0
        if "documents" not in kw:
            assert taken.sum() <= 128 * steps.sum()


def test_rows_that_attend_nothing_have_an_item():
    plan = _plan([300, 2], [300, 9], mask=np.zeros((302, 4), dtype=np.int64))
    rows = {(x[0], x[1], x[3]) for x in plan.host_items.tolist() if x[0] >= 0}
    assert rows == {(0, h, r) for h in range(2) for r in range(0, 900, 256)} | {(1, 0, 0), (1, 1, 0)}
    assert plan.n_merges == 0


def test_a_batch_that_waits():
    plan = _plan([0, 0], [5, 0], mask=ChunkMask(window=3, documents=[[0, 2], []]))
    assert plan.n_items == plan.n_tokens == 0 and plan.ranges.shape == (0, 4)
    assert _plan([0, 0], [5, 0], mask=np.zeros((0, 4), dtype=np.int32)).n_items == 0


def test_an_empty_mask_is_the_causal_plan():
    a, b = _plan([700, 1], [900, 5000]), _plan([700, 1], [900, 5000], mask=ChunkMask())
    assert b.ranges is None and np.array_equal(a.host_items, b.host_items) and np.array_equal(a.host_merges, b.host_merges)
    c = _plan([700, 1], [900, 5000], mask=ChunkMask(window=5000))
    assert np.array_equal(a.host_items, c.host_items) and np.all(c.host_gaps == -1)


def test_mask_refusals():
    for kw in (dict(window=0), dict(window=-3), dict(window=1.5), dict(window=True), dict(window=2 ** 31), dict(sinks=2), dict(window=4, sinks=-1),
               dict(prefix=-1), dict(prefix=[3, -1]), dict(prefix=2.0), dict(documents=[[1]]), dict(documents=[[0, 5, 5]]), dict(documents=[[0, 7, 5]]),
               dict(documents=[[0, 2.5]])):
        with pytest.raises(ValueError):
            ChunkMask(**kw)
    for kw in (dict(prefix=11), dict(prefix=(3, 3, 3)), dict(prefix=(3,)), dict(documents=[[0]]), dict(documents=[[0, 10], [0]])):
        with pytest.raises(ValueError):
            _plan([4, 2], [10, 20], mask=ChunkMask(**kw))
    for bad in (np.zeros((5, 4), dtype=np.int32), np.zeros((6, 4)), np.full((6, 4), -1), np.full((6, 4), 2 ** 33), np.tile([0, 0, 0, 11], (6, 1)),
                np.tile([3, 2, 0, 0], (6, 1)), "causal"):
        with pytest.raises(ValueError):
            _plan([4, 2], [10, 20], mask=bad)
    with pytest.raises(ValueError):
        ChunkMask().ranges([3], [2])


def test_call_refusals():
    kp, vp = _pools()
    plan = plan_chunk(kp, vp, [2], [20], kv_heads=2, q_per_kv=3, mask=ChunkMask(window=4))
    table = torch.zeros((1, 2, 2), dtype=torch.int32)
    q = torch.zeros((2, 6, 64))
    for kw in (dict(cap=0.0), dict(cap=-2.0), dict(cap=float("inf")), dict(cap=float("nan")), dict(slopes=torch.zeros(5)),
               dict(slopes=torch.zeros(6, dtype=torch.float64)), dict(slopes=torch.zeros(6, 2)[:, 0]), dict(slopes=torch.zeros(1, 6))):
        with pytest.raises(ValueError):
            attend_chunk(kp, table, vp, table, q, plan, **kw)


def test_entry_refusals():
    """The C entries' own checks (nothing is launched)."""
    import ctypes as C

    L = _lib.lib()
    n = np.array([2], dtype=np.int32)
    counts = [C.c_int32() for _ in range(5)]

    def plan(ranges, gaps=None, most=0):
        return L.dc_plan_chunk_ranges(n.ctypes.data, n.ctypes.data, None if ranges is None else ranges.ctypes.data, 1, 1, 1, 64, 8, 128,
                                      None, gaps, most, *(C.byref(c) for c in counts[:3]), None, 0, *(C.byref(c) for c in counts[3:]))

    assert plan(None) == _lib.DC_EINVAL
    assert plan(np.zeros((2, 4), dtype=np.int32), None, 4) == _lib.DC_EINVAL
    assert plan(np.array([[0, 3, 0, 0], [0, 0, 0, 0]], dtype=np.int32)) == _lib.DC_EINVAL
    assert plan(np.array([[0, 2, 0, 0], [0, 0, 0, 0]], dtype=np.int32)) == _lib.DC_ESPACE and counts[0].value == 1

    def call(**kw):
        pool = _lib.Pool(1 << 20, 1 << 20, 1 << 20, 1, _lib.geometry(64, 32, 16), 1)
        rows = _lib.TokenRows(1 << 20, 64, 64, 1, _lib.DT_F16)
        rule = _lib.ScoreRule(kw.get("cap", 0.0), None, kw.get("ranges"), kw.get("gaps"))
        return L.dc_attend_chunk_rule(pool, pool, 1 << 20, 1 << 20, 1, 1 << 20, 1, 0, 0, None, 0, 0, 1, 1, 1, rows, kw.get("scale", 1.0), rule,
                                      rows, None, 0, None)

    for kw in (dict(cap=-1.0), dict(cap=float("nan")), dict(cap=float("inf")), dict(cap=1e-30, scale=1e30), dict(ranges=1 << 20 | 8),
               dict(ranges=1 << 20, gaps=1 << 20 | 4), dict(gaps=1 << 20)):
        assert call(**kw) == _lib.DC_EINVAL, kw
