"""2- and 3-bit pages of one pool written by one call: rows of both widths, and
of others, next to each other in a wavefront."""
import numpy as np
import pytest

from tests.test_gpu_rotary import _dense, _form, _oracle_page, _same

pytestmark = pytest.mark.gpu


def _pages(hd, gs, P, names, n):
    """``n`` pages for each of ``names`` in one pool, ids in turn."""
    from dotcache_amd.page_pool import DevicePagePool, PoolGeometry

    pool = DevicePagePool(PoolGeometry(hd, gs, P), reserve_bytes=1 << 18, reserve_pages=64)
    return pool, np.stack([pool.allocate(*_form(f), n, tokens=P) for f in names], axis=1).ravel(), list(names) * n


@pytest.mark.parametrize("hd,gs", [(128, 32), (64, 32), (256, 64), (96, 32), (64, 16), (40, 8)])
@pytest.mark.parametrize("names", [("a3", "a2"), ("s2", "a3"), ("s3", "a4", "a2"), ("m3", "a2", "s3", "s8")])
def test_widths_side_by_side(hd, gs, names):
    """Token t of every page in turn: neighbouring rows have other widths."""
    import torch

    P, n = 4, 3
    print(f"narrow pages {hd} {gs} {names}", flush=True)
    rng = np.random.default_rng(hd)
    pool, ids, form = _pages(hd, gs, P, names, n)
    vpool, vids, vform = _pages(hd, gs, P, tuple(reversed(names)), n)
    W = len(ids)
    x = rng.normal(size=(2, W, P, hd)).astype(np.float32)
    # rows (t, page): encode_rows, then the same as tokens of one head of W sequences of one page
    turn = np.ascontiguousarray(x.transpose(0, 2, 1, 3).reshape(2, P * W, hd))
    slot, at = np.repeat(np.arange(P), W), np.tile(np.arange(W), P)
    rows = torch.from_numpy(turn).cuda()
    tables = torch.from_numpy(np.stack([ids, vids]).astype(np.int32).reshape(2, W, 1, 1)).cuda()

    def check():
        got = pool.read_tokens_with(vpool, tables, at, slot)
        for i, (p, pid, names_of) in enumerate(((pool, ids, form), (vpool, vids, vform))):
            for w in range(W):
                want = _oracle_page(x[i, w], names_of[w], hd, gs, "KV"[i])
                _same(p.download_page(pid[w], kind="KV"[i]), want, np.arange(P))
                assert np.array_equal(got[i][torch.from_numpy(np.flatnonzero(at == w)).cuda(), 0].cpu().numpy(), _dense(names_of[w], want))

    pool.encode_rows(rows[0], ids[at], slot.astype(np.int32))
    vpool.encode_rows(rows[1], vids[at], slot.astype(np.int32))
    check()
    for p in (pool, vpool):
        p.arena.fill_(0xAB)
    pool.append_rotary_with(vpool, None, rows[0][:, None], rows[1][:, None], None, None, tables, at, slot)
    check()
