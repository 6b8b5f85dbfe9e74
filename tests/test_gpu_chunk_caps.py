"""Caps of the chunk attention from far below the scores to far above them: a
capped score is off by a share of itself, not of the cap."""
import numpy as np
import pytest

from tests.test_gpu_chunk import _Batch, _dt

pytestmark = pytest.mark.gpu


def _check(batch, new, n_q, dtype, cap, size, rng, **kw):
    """Against fp64, causal.  A logit q . k is off by hd + 4 products and sums of 2^-24
    each (16-bit queries: operands rounded to fp16, 2^-10 of the terms); the cap's slope is at most 1, and its
    own arithmetic is off by 2^-20 of the capped score, relative: a polynomial to a rounding of
    2^-24 each in six steps, or 1 - 2 / (e + 1) with e from 1 on, where the quotient, off by
    2^-22.4 (exponential and reciprocal 2^-23 each, their argument and sum 2^-24), is taken from 1 and leaves tanh(1/2) at least: 2^-21.3.
    Exponentials 2^-22.  From there on weights and values as everywhere: a weight
    off by e^2delta - 1, their sum by the mean of that, (16 bits) one rounding of 2^-11 each, weights below
    fp16's range 2^-25 of the largest, (fp32) sums of 2^-24 a token; then the output's own rounding."""
    import torch

    hd, T = batch.hd, sum(new)
    q = torch.from_numpy((rng.normal(size=(T, batch.H * n_q, hd)) * size).astype(np.float32)).to(_dt(dtype)).cuda()
    scale = 1.0 / np.sqrt(hd)
    got = batch.attend(q, batch.plan(new, n_q), scale, cap=cap, **kw).double().cpu().numpy()
    qd, t0, most = q.double().cpu().numpy(), 0, 0.0
    per = (hd + 4) * 2.0 ** -24 if dtype == "f32" else 2.0 ** -10
    half = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
    for b, n in enumerate(new):
        c = batch.ctx[b]
        ok = np.arange(c)[None, :] <= np.arange(c - n, c)[:, None]
        for j in range(batch.H * n_q):
            k, v = (x[b, j // n_q, :c] for x in batch.rows)
            s = scale * (qd[t0: t0 + n, j] @ k.T)
            delta = per * scale * (np.abs(qd[t0: t0 + n, j]) @ np.abs(k).T)
            s = cap * np.tanh(s / cap)
            delta = delta + 2.0 ** -20 * np.abs(s) + 2.0 ** -22
            s = np.where(ok, s, -np.inf)
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            want, e = p @ v, np.expm1(2 * np.where(ok, delta, 0.0))
            own = (c + 8) * 2.0 ** -24 if dtype == "f32" else 2.0 ** -10 * (1 + 2.0 ** -6)
            low = 0.0 if dtype == "f32" else c * 2.0 ** -25 * np.abs(v).max()
            bound = (p * e) @ np.abs(v) + ((p * e).sum(1, keepdims=True) + own) * (p @ np.abs(v)) + low + half * np.abs(want)
            most = max(most, float(np.max(np.abs(got[t0: t0 + n, j] - want) / bound)))
        t0 += n
    assert most <= 1.0, most


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cap", [0.5, 5.0, 50.0, 1e3, 1e6, 1e8, 1e30])
def test_caps_of_any_size(cap, dtype):
    """Row tiles, drafted tokens and a decode; scores of order 1, and of order 10."""
    for hd in (64, 128, 256):
        for size in (0.5, 4.0):
            print(f"chunk cap {cap} {dtype} {hd} {size}", flush=True)
            rng = np.random.default_rng(hd)
            batch = _Batch(rng, [260, 150, 40], 1, hd, 32, "a4", "s4")
            _check(batch, [120, 3, 1], 3, dtype, cap, size, rng)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_caps_on_the_general_kernel(dtype):
    """2-bit pages and a head_dim of no whole groups."""
    for cap in (3.0, 50.0, 1e6):
        print(f"chunk cap general {cap} {dtype}", flush=True)
        rng = np.random.default_rng(4)
        _check(_Batch(rng, [200, 90], 2, 80, 16, "a2", "s4", (16, 32)), [90, 2], 2, dtype, cap, 1.0, rng)


def test_one_score_by_itself():
    """Two tokens, a key of zeros with a value of 0 and one with 1: the output
    is the logistic function of the capped score, which fp32 shows to 2^-24."""
    import torch

    from dotcache_amd.chunk import attend_chunk, plan_chunk
    from dotcache_amd.page_pool import DevicePagePool, PoolGeometry

    pools = [DevicePagePool(PoolGeometry(64, 32, 16), reserve_bytes=1 << 16, reserve_pages=16) for _ in range(2)]
    ids = [p.allocate(0, 0, 1, tokens=2) for p in pools]
    rows = torch.zeros(2, 64, device="cuda")
    rows[1] = 1.0
    for p, i in zip(pools, ids):
        p.encode_rows(rows / 64 if p is pools[0] else rows, np.repeat(i, 2).astype(np.int32), np.arange(2, dtype=np.int32))
    tables = [torch.from_numpy(i.reshape(1, 1, 1).astype(np.int32)).cuda() for i in ids]
    want_s = np.concatenate([np.linspace(-9, 9, 181), np.array([0.5, -0.5, 1.0, -1.0]) * 3.0])
    for cap in (3.0, 6.0, 50.0, 1e4, 1e7):
        s = want_s.astype(np.float32)
        # (64 equal products of s / 64: the score is s, exactly); every score a sequence of its own
        q = torch.from_numpy(np.repeat(s[:, None, None], 64, axis=2)).cuda()
        plan = plan_chunk(*pools, [1] * s.size, [2] * s.size, kv_heads=1, q_per_kv=1)
        k_table, v_table = (t.expand(s.size, 1, 1).contiguous() for t in tables)
        got = attend_chunk(pools[0], k_table, pools[1], v_table, q, plan, cap=cap).double().cpu().numpy()[:, 0]
        x = cap * np.tanh(s.astype(np.float64) / cap)
        want = 1.0 / (1.0 + np.exp(-x))
        # slope p (1 - p) of the score's 2^-20; exponential, sum and quotient 2^-22
        bound = want * (1 - want) * 2.0 ** -20 * np.abs(x) + 2.0 ** -21 * want
        assert np.all(np.abs(got - want[:, None]) <= bound[:, None]), (cap, float(np.max(np.abs(got - want[:, None]) / bound[:, None])))


def test_caps_and_scores_near_the_end_of_fp32():
    """Scores of 10^38 under a cap of 2 x 10^38, twice which fp32 does not hold:
    the token of the largest has all the weight, whatever its score's sign or share of the cap."""
    import torch

    from dotcache_amd.chunk import attend_chunk, plan_chunk
    from dotcache_amd.page_pool import DevicePagePool, PoolGeometry

    pools = [DevicePagePool(PoolGeometry(64, 32, 16), reserve_bytes=1 << 16, reserve_pages=16) for _ in range(2)]
    ids = [p.allocate(0, 0, 1, tokens=4) for p in pools]
    keys = torch.tensor([0.25, -0.5, 1.0, 0.5], device="cuda")[:, None].expand(4, 64).contiguous()
    values = torch.arange(1.0, 5.0, device="cuda")[:, None].expand(4, 64).contiguous()
    for p, i, rows in zip(pools, ids, (keys, values)):
        p.encode_rows(rows, np.repeat(i, 4).astype(np.int32), np.arange(4, dtype=np.int32))
    tables = [torch.from_numpy(i.reshape(1, 1, 1).astype(np.int32)).cuda() for i in ids]
    plan = plan_chunk(*pools, [1], [4], kv_heads=1, q_per_kv=1)
    for sign, want in ((1.0, 3.0), (-1.0, 2.0)):
        q = torch.full((1, 1, 64), sign * 2.0 ** 120, device="cuda")
        # 64 x 2^120 = 2^126 (8.5e37) under the largest key; the scale takes it to a quarter, once and twice that
        for scale in (0.25, 1.0, 2.0):
            got = attend_chunk(pools[0], tables[0], pools[1], tables[1], q, plan, query_scale=scale, cap=2e38)
            assert bool((got == want).all()), (sign, scale, got.flatten()[:4])
