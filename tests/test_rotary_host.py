"""Refusals of the norm-and-rotate entry points, on the CPU: nothing here
reaches a GPU."""
import ctypes as C

import numpy as np
import pytest
import torch

from dotcache_amd import _lib
from dotcache_amd.page_pool import DevicePagePool, PoolGeometry
from dotcache_amd.rotary import RotaryTable, index_tensor, norm_rotate


def _table(hd=64, n=32, **kw):
    return RotaryTable(hd, n, device="cpu", **kw)


def test_table_values_and_refusals():
    t = _table(8, 5, rotary_dim=4, base=100.0, amplitude=2.0).table.numpy()
    a = np.arange(5)[:, None] * np.array([1.0, 0.1])
    np.testing.assert_allclose(t, 2 * np.concatenate([np.cos(a), np.sin(a)], axis=1), rtol=2.0 ** -23, atol=0)
    for bad in (dict(rotary_dim=3), dict(rotary_dim=10), dict(rotary_dim=0), dict(inv_freq=[1.0])):
        with pytest.raises(ValueError):
            _table(8, 5, **bad)
    with pytest.raises(ValueError):
        _table(8, 0)


def test_norm_rotate_refusals():
    q, k, pos = torch.zeros(4, 3, 64), torch.zeros(4, 1, 64), torch.zeros(4, dtype=torch.int32)
    t = _table()
    bad = [dict(queries=None, keys=None), dict(keys=k[:3]), dict(keys=k.half()), dict(positions=pos[:3]),
           dict(positions=pos.float()), dict(positions=[0, 1, 2, 32]), dict(positions=np.array([0, -1, 2, 3])),
           dict(rotary=_table(32)), dict(q_weight=torch.ones(32)), dict(k_weight=torch.ones(2, 64)),
           dict(q_weight=torch.ones(64), eps=-1.0), dict(q_weight=torch.ones(64), eps=float("nan")),
           dict(q_weight=torch.ones(64, dtype=torch.int32)), dict(queries=q.transpose(1, 2)), dict(queries=q[0]),
           dict(queries=q.double(), keys=None), dict(out=(q, None)), dict(out=(q.half(), k)), dict(out=(q[:3], k)),
           dict(queries=q[:, :0], keys=None)]
    for change in bad:
        args = dict(queries=q, keys=k, positions=pos, rotary=t) | change
        with pytest.raises(ValueError):
            norm_rotate(args.pop("queries"), args.pop("keys"), args.pop("positions"), args.pop("rotary"), **args)
    with pytest.raises(ValueError, match="GPU"):  # all in order, but not on a GPU
        norm_rotate(q, k, pos, t)


def test_append_and_read_refusals():
    geo = PoolGeometry(64, 32, 16)
    kp, vp = (DevicePagePool(geo, device="cpu", reserve_bytes=1 << 16, reserve_pages=16) for _ in range(2))
    for p in (kp, vp):
        p.allocate(1, 4, 4, tokens=16)
    tables = torch.arange(4, dtype=torch.int32).reshape(1, 2, 1, 2).repeat(2, 1, 1, 1)
    x, t = torch.zeros(3, 1, 64), _table()
    idx = torch.zeros(3, dtype=torch.int32)
    other = DevicePagePool(PoolGeometry(64, 32, 32), device="cpu", reserve_bytes=1 << 16, reserve_pages=16)
    good = dict(v_pool=vp, queries=x, keys=x, values=x, positions=idx, rotary=t, tables=tables, row=idx, token=idx)
    bad = [dict(v_pool=other), dict(queries=x[:2]), dict(queries=x.half()), dict(keys=x.repeat(1, 2, 1)), dict(values=x.half()),
           dict(values=x[..., :32]), dict(positions=idx[:2]), dict(positions=[0, 1, 99]), dict(rotary=_table(32)),
           dict(tables=tables.long()), dict(tables=tables[0]), dict(tables=tables[:, :0]), dict(tables=tables.transpose(1, 3)),
           dict(row=idx[:2]), dict(token=idx[:2]), dict(token=idx.float()), dict(token=[0.5, 1, 2]), dict(k_weight=torch.ones(3)),
           dict(out=x[:2]), dict(out=x.bfloat16()), dict(keep=(torch.zeros(4, 64), torch.zeros(4, 64), idx[:1], 1)),
           dict(keep=(torch.zeros(4, 64), torch.zeros(5, 64), idx, 1)), dict(keep=(torch.zeros(4, 64).half(),) * 2 + (idx, 1))]
    for change in bad:
        args = good | change
        with pytest.raises(ValueError):
            kp.append_rotary_with(**args)
    for change in (dict(v_pool=other), dict(tables=tables.long()), dict(token=idx[:2]), dict(dtype=torch.float64),
                   dict(out=(x, x.half())), dict(out=(x, x), dtype=torch.float16), dict(out=(x[:2], x))):
        args = dict(v_pool=vp, tables=tables, row=idx, token=idx) | change
        with pytest.raises(ValueError):
            kp.read_tokens_with(**args)


def test_host_indexes_fit_32_bits():
    for bad in ([2 ** 40], torch.tensor([-2 ** 33])):
        with pytest.raises(ValueError):
            index_tensor(bad, "token", 1, torch.device("cpu"))
    assert index_tensor([5], "token", 1, torch.device("cpu")).dtype == torch.int32


def test_c_entry_refusals():
    """The C entries refuse bad arguments before any launch (pointers here are never read)."""
    lib = _lib.lib()
    p, rows = 4096, lambda **kw: _lib.TokenRows(**(dict(data=4096, token_stride=64, head_stride=64, n_heads=1, dtype=0) | kw))  # noqa: E731
    none, norm = _lib.TokenRows(), _lib.Norm()
    rot = lambda **kw: _lib.Rotary(**(dict(table=4096, n_positions=8, rotary_dim=64, interleaved=0) | kw))  # noqa: E731

    def nr(n=1, hd=64, pos=p, rotary=rot(), q=rows(), qn=norm, qo=rows(), k=none, kn=norm, ko=none):
        return lib.dc_norm_rotate(n, hd, pos, rotary, q, qn, qo, k, kn, ko, None)

    assert nr(n=0) == _lib.DC_OK
    for bad in (dict(n=-1), dict(hd=0), dict(hd=9000), dict(rotary=rot(rotary_dim=65)), dict(rotary=rot(rotary_dim=66)),
                dict(rotary=rot(rotary_dim=-2)), dict(pos=None), dict(rotary=rot(table=None)), dict(rotary=rot(table=4100)),
                dict(rotary=rot(n_positions=0)), dict(q=none), dict(q=rows(dtype=5)), dict(q=rows(data=None)),
                dict(qo=rows(n_heads=2)), dict(qo=rows(data=None)), dict(k=rows(dtype=1), ko=rows()),
                dict(qn=_lib.Norm(4096, 9, 0, 1e-6)), dict(qn=_lib.Norm(4096, 0, 0, -1.0)), dict(n=2 ** 33)):
        assert nr(**bad) == _lib.DC_EINVAL, bad

    geo = _lib.geometry(64, 32, 16)
    pool = lambda **kw: _lib.Pool(**(dict(arena=4096, arena_bytes=1 << 20, descs=4096, n_descs=4, geometry=geo) | kw))  # noqa: E731
    dest = lambda **kw: _lib.TokenDest(**(dict(k_pages=4096, v_pages=4096, row=4096, token=4096, n_rows=1, n_pages=1, page_tokens=16) | kw))  # noqa: E731

    def ap(n=0, pos=p, rotary=rot(), q=rows(), qo=rows(), k=rows(), v=rows(), d=dest(), kp=pool(), vp=pool(), keep=(None, None, None, 0, 0)):
        return lib.dc_append_rotary(n, pos, rotary, q, norm, qo, k, norm, v, d, kp, vp, *keep, None)

    assert ap() == _lib.DC_OK and ap(q=none, qo=none) == _lib.DC_OK
    for bad in (dict(n=-1), dict(kp=pool(arena=None)), dict(vp=pool(n_descs=0)), dict(kp=pool(geometry=_lib.geometry(32, 32, 16))),
                dict(d=dest(row=None)), dict(d=dest(n_rows=0)), dict(d=dest(page_tokens=17)), dict(d=dest(page_tokens=0)),
                dict(k=rows(n_heads=2)), dict(v=rows(dtype=1)), dict(q=rows(dtype=1), qo=rows(dtype=1)), dict(qo=none),
                dict(keep=(4096, None, 4096, 0, 1)), dict(keep=(4096, 4096, None, 0, 1)), dict(keep=(4100, 4096, 4096, 0, 1))):
        assert ap(**bad) == _lib.DC_EINVAL, bad

    def rd(n=0, d=dest(), kp=pool(), vp=pool(), ko=rows(), vo=rows()):
        return lib.dc_read_tokens(n, d, kp, vp, ko, vo, None)

    assert rd() == _lib.DC_OK
    for bad in (dict(n=-1), dict(ko=none), dict(vo=rows(n_heads=2)), dict(vo=rows(dtype=7)), dict(d=dest(page_tokens=17)),
                dict(d=dest(token=None)), dict(d=dest(n_pages=0)), dict(vp=pool(geometry=_lib.geometry(32, 32, 16))), dict(kp=pool(descs=None))):
        assert rd(**bad) == _lib.DC_EINVAL, bad
    assert C.sizeof(_lib.TokenRows) == 32 and C.sizeof(_lib.TokenDest) == 48
