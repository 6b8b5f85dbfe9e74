"""The chunk attention's planner and refusals, on the CPU."""
import ctypes as C

import numpy as np
import pytest
import torch

from dotcache_amd import _lib
from dotcache_amd.chunk import attend_chunk, plan_chunk, workspace_bytes
from dotcache_amd.page_pool import DevicePagePool, PoolGeometry


def _pools(hd=64, P=16, n=8):
    pools = [DevicePagePool(PoolGeometry(hd, 32, P), device="cpu", reserve_bytes=1 << 16, reserve_pages=16) for _ in range(2)]
    for p in pools:
        p.allocate(1, 4, n, tokens=P)
    return pools


def _plan(new, ctx, H=2, n_q=3, **kw):
    return plan_chunk(*_pools(), new, ctx, kv_heads=H, q_per_kv=n_q, **kw)


@pytest.mark.parametrize("new,ctx", [([1], [1]), ([0, 5], [0, 5]), ([700, 1, 0, 43], [900, 5000, 77, 43]), ([1] * 64, list(range(1, 65))),
                                     ([3000], [100000])])
@pytest.mark.parametrize("target", [1, 37, 512])
def test_items_cover_every_row_and_token_once(new, ctx, target):
    H, n_q = 2, 3
    plan = _plan(new, ctx, H, n_q, target_items=target)
    start = np.concatenate([[0], np.cumsum(new)])
    items = [dict(zip(_lib.CHUNK_ITEM_FIELDS, x)) for x in plan.host_items.tolist()]
    assert all(x["row_end"] <= plan.few_rows <= 64 for x in items[: plan.n_few])
    assert all(x["row_end"] - x["row_begin"] > 64 or x["row_begin"] > 0 for x in items[plan.n_few:] if x["seq"] >= 0)
    items = [x for x in items if x["seq"] >= 0]
    seen, slots = {}, set()
    for x in items:
        b = x["seq"]
        assert 0 <= x["kv_head"] < H and x["q_begin"] == start[b] and x["first"] == ctx[b] - new[b]
        assert x["row_begin"] % 256 == 0 and x["row_end"] == min(x["row_begin"] + 256, new[b] * n_q)
        n_rows = x["row_end"] - x["row_begin"]
        seen.setdefault((b, x["kv_head"], x["row_begin"]), []).append((x["kv_begin"], x["kv_end"], x["partial"]))
        if x["partial"] >= 0:
            mine = set(range(x["partial"], x["partial"] + n_rows))
            assert max(mine) < plan.n_partials and not mine & slots
            slots |= mine
    assert len(slots) == plan.n_partials
    assert len(seen) == sum(-(-n * n_q // 256) for n in new) * H
    merges = {(h, q, r): (p, n) for h, q, r, _, p, n in plan.host_merges.tolist()}
    for (b, h, r), parts in seen.items():
        parts.sort()
        last = ctx[b] - new[b] + (min(r + 256, new[b] * n_q) - 1) // n_q
        assert parts[0][0] == 0 and parts[-1][1] == last + 1
        assert all(x[1] == y[0] for x, y in zip(parts, parts[1:])) and all(x[0] % 128 == 0 and x[1] > x[0] for x in parts)
        if len(parts) == 1:
            assert parts[0][2] == -1
        else:
            assert merges[h, int(start[b]), r] == (parts[0][2], len(parts))
            rows = min(256, new[b] * n_q - r)
            assert [x[2] for x in parts] == list(range(parts[0][2], parts[0][2] + rows * len(parts), rows))
    assert len(merges) == sum(len(x) > 1 for x in seen.values()) == plan.n_merges
    assert plan.n_tokens == sum(new) and workspace_bytes(plan, 64) == plan.n_partials * 66 * 4


def test_equal_work_on_every_die():
    """Consecutive items go to consecutive dies: each takes an equal share."""
    plan = _plan([2048, 3], [16384, 20000], 4, 7, target_items=512)
    length = plan.host_items[:, 7] - plan.host_items[:, 6]
    assert 0 < plan.n_few < plan.n_items and plan.few_rows == 21
    for part in (length[: plan.n_few], length[plan.n_few:]):
        share = [int(part[i::8].sum()) for i in range(8)]
        assert max(share) - min(share) <= 2 * int(part.max())


def test_plan_refusals():
    for args in (dict(new=[], ctx=[]), dict(new=[1], ctx=[1, 2]), dict(new=[3], ctx=[2]), dict(new=[-1], ctx=[2]), dict(new=[1.5], ctx=[2]),
                 dict(new=[[1]], ctx=[[2]]), dict(new=[1], ctx=[2 ** 31]), dict(new=[1], ctx=[1], H=0), dict(new=[1], ctx=[1], n_q=0),
                 dict(new=[1], ctx=[1], target_items=0), dict(new=[2 ** 30], ctx=[2 ** 30])):
        with pytest.raises(ValueError):
            _plan(args.pop("new"), args.pop("ctx"), **args)
    with pytest.raises(ValueError):
        plan_chunk(*_pools(hd=320), [1], [1], kv_heads=1, q_per_kv=1)
    with pytest.raises(ValueError):
        plan_chunk(_pools()[0], _pools(P=32)[0], [1], [1], kv_heads=1, q_per_kv=1)
    n = np.ones(1, dtype=np.int32)
    c = [C.c_int32() for _ in range(5)]
    tail = (*(C.byref(x) for x in c[:3]), None, 0, C.byref(c[3]), C.byref(c[4]))
    plan = _lib.lib().dc_plan_chunk
    assert plan(n.ctypes.data, n.ctypes.data, 1, 2, 3, 64, 8, 256, None, 0, *tail) == _lib.DC_ESPACE and c[0].value >= 2
    assert plan(None, n.ctypes.data, 1, 2, 3, 64, 8, 256, None, 0, *tail) == _lib.DC_EINVAL
    assert plan(n.ctypes.data, n.ctypes.data, 1, 2, 3, 64, 8, 0, None, 0, *tail) == _lib.DC_EINVAL
    assert plan(n.ctypes.data, n.ctypes.data, 1, 2, 3, 0, 8, 256, None, 0, *tail) == _lib.DC_EINVAL


def test_attend_refusals():
    pools = _pools()
    plan = plan_chunk(*pools, [4, 2], [30, 2], kv_heads=1, q_per_kv=2)
    table = torch.zeros(2, 1, 2, dtype=torch.int32)
    q = torch.zeros(6, 2, 64)
    good = dict(pool=pools[0], k_table=table, v_pool=pools[1], v_table=table, queries=q, plan=plan)
    for change in (dict(k_table=table[0]), dict(k_table=table[:1]), dict(v_table=table[:, :, :1]), dict(k_table=table.long(), v_table=table.long()),
                   dict(k_table=table[:, :, :1], v_table=table[:, :, :1]), dict(queries=q[:5]), dict(queries=q[:, :1]), dict(queries=q[..., :32]),
                   dict(queries=q.double()), dict(queries=q.repeat(2, 1, 1)), dict(out=q[:5]), dict(out=q.half()), dict(queries=q.transpose(0, 2)),
                   dict(v_pool=_pools(P=32)[0]), dict(v_pool=_pools(hd=32)[0])):
        with pytest.raises(ValueError):
            attend_chunk(**(good | change))
    with pytest.raises(ValueError, match="GPU"):
        attend_chunk(**good)
    split = plan_chunk(*_pools(P=16), [1], [6000], kv_heads=1, q_per_kv=1)
    assert split.n_partials > 0
    wide = torch.zeros(1, 1, 375, dtype=torch.int32)
    with pytest.raises(ValueError, match="workspace"):
        attend_chunk(pools[0], wide, pools[1], wide, torch.zeros(1, 1, 64), split, workspace=torch.zeros(16, dtype=torch.uint8))


def test_c_entry_refusals():
    """Refused before any launch (pointers here are never read)."""
    geo = _lib.geometry(64, 32, 16)
    pool = lambda **kw: _lib.Pool(**(dict(arena=4096, arena_bytes=1 << 20, descs=4096, n_descs=4, geometry=geo) | kw))  # noqa: E731
    rows = lambda **kw: _lib.TokenRows(**(dict(data=4096, token_stride=64, head_stride=64, n_heads=2, dtype=1) | kw))  # noqa: E731

    def go(kp=pool(), vp=pool(), kt=4096, vt=4096, stride=1, items=4096, n_items=0, few=0, few_rows=0, merges=None, n_merges=0, parts=0, B=1, H=1, T=1,
           q=rows(), out=rows(), ws=None, size=0):
        return _lib.lib().dc_attend_chunk(kp, vp, kt, vt, stride, items, n_items, few, few_rows, merges, n_merges, parts, B, H, T, q, 1.0, out, ws, size, None)

    assert go() == _lib.DC_OK
    for bad in (dict(kp=pool(geometry=_lib.geometry(512, 32, 16)), vp=pool(geometry=_lib.geometry(512, 32, 16))),
                dict(vp=pool(geometry=_lib.geometry(32, 32, 16))), dict(vp=pool(geometry=_lib.geometry(64, 32, 32))), dict(n_items=-1),
                dict(B=0), dict(stride=0), dict(n_items=1, kt=None), dict(n_items=1, items=None), dict(n_items=1, n_merges=1),
                dict(n_items=1, q=rows(dtype=4)), dict(n_items=1, out=rows(dtype=0)), dict(n_items=1, out=rows(n_heads=1)),
                dict(n_items=1, H=3), dict(n_items=1, few=2, few_rows=1), dict(n_items=1, few=1), dict(n_items=1, few=1, few_rows=65), dict(few=-1), dict(n_items=1, kp=pool(descs=None))):
        assert go(**bad) == _lib.DC_EINVAL, bad
    assert go(n_items=1, parts=1, ws=4096, size=16) == _lib.DC_ESPACE
    assert go(n_items=1, parts=1, ws=None, size=1 << 20) == _lib.DC_ESPACE


def test_long_contexts_are_refused():
    with pytest.raises(ValueError, match="too long a context"):
        _plan([1], [2 ** 31 - 65536])
    assert _plan([1], [2 ** 31 - 65537], target_items=4).n_items > 0


@pytest.mark.parametrize("new,ctx,H,n_q", [([2048, 2048], [16384, 16384], 4, 7), ([5, 5, 5, 5], [131000, 60000, 3000, 900], 4, 7),
                                           ([700, 1, 333, 64, 512], [8192, 5000, 900, 4097, 700], 4, 4)])
def test_work_is_spread_over_the_card(new, ctx, H, n_q):
    """Blocks start in order, each on the first free slot of its die: the last is
    done within a quarter of an even share, or within the longest part."""
    plan = _plan(new, ctx, H, n_q, target_items=256)
    for part, slots in ((plan.host_items[: plan.n_few], 512), (plan.host_items[plan.n_few:], 256)):
        length = np.where(part[:, 0] >= 0, part[:, 7] - part[:, 6], 0)
        if not length.any():
            continue
        done = 0
        for die in range(8):
            free = np.zeros(slots // 8, dtype=np.int64)
            for n in length[die::8]:
                free[np.argmin(free)] += n
            done = max(done, int(free.max()))
        assert done <= max(1.25 * length.sum() / slots, length.max())
