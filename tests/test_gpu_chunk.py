"""Chunk attention over compressed pages against fp64 numpy on the pages' own
values: every page format, odd head_dims and page sizes, shared heads, ragged
batches with waiting sequences, split ranges, strided and padded queries,
tokens without a page, and values that are not finite where a row does not
look."""
import numpy as np
import pytest

from tests.test_gpu_rotary import _form

pytestmark = pytest.mark.gpu


def _dt(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


class _Batch:
    """Sequences of ``ctx`` tokens in two pools, their pages scattered; the
    last page of each exact where ``tail``."""

    def __init__(self, rng, ctx, H, hd, P, key="a4", value="s4", gs=(32, 32), tail=True, layout="group_major", spare=0):
        import torch

        from dotcache_amd.page_pool import DevicePagePool, PoolGeometry

        B, W = len(ctx), max(-(-max(ctx) // P), 1) + spare
        self.ctx, self.P, self.H, self.hd = ctx, P, H, hd
        self.pools, self.host, self.tables, self.rows = [], [], [], []
        for name, g in ((key, gs[0]), (value, gs[1])):
            pool = DevicePagePool(PoolGeometry(hd, g, P, layout), reserve_bytes=1 << 20, reserve_pages=64)
            table = rng.permutation(pool.allocate(*_form(name), B * H * W, tokens=P)).reshape(B, H, W).astype(np.int32)
            for b, n in enumerate(ctx):
                if n == 0:
                    continue
                last = (n - 1) // P
                if tail:
                    table[b, :, last] = pool.allocate(0, 0, H)
                pool.set_tokens(table[b, :, last], n - last * P)
            x = rng.normal(size=(B, H, W * P, hd)).astype(np.float32) * np.exp(0.5 * rng.normal(size=(1, H, 1, hd))).astype(np.float32)
            t = np.arange(W * P)
            pool.encode_rows(torch.from_numpy(x.reshape(-1, hd)).cuda(), np.ascontiguousarray(table[:, :, t // P]).reshape(-1),
                             np.broadcast_to(t % P, (B, H, W * P)).reshape(-1).astype(np.int32))
            self.pools.append(pool)
            self.host.append(table)
            self.tables.append(torch.from_numpy(table).cuda())
        self.read()

    def read(self):
        """The pages' values, [B, H, tokens, hd] fp64, keys and values."""
        import torch

        B, H, W = self.host[0].shape
        T = W * self.P
        both = torch.stack(self.tables).contiguous()
        got = self.pools[0].read_tokens_with(self.pools[1], both, np.repeat(np.arange(B), T), np.tile(np.arange(T), B))
        self.rows = [y.reshape(B, T, H, self.hd).transpose(1, 2).cpu().numpy().astype(np.float64) for y in got]

    def plan(self, new, n_q, **kw):
        from dotcache_amd.chunk import plan_chunk

        return plan_chunk(*self.pools, new, self.ctx, kv_heads=self.H, q_per_kv=n_q, **kw)

    def attend(self, q, plan, scale, **kw):
        from dotcache_amd.chunk import attend_chunk

        return attend_chunk(self.pools[0], self.tables[0], self.pools[1], self.tables[1], q, plan, query_scale=scale, **kw)


def _want(batch, q, new, n_q, scale):
    """fp64 outputs [tokens, Hq, hd] and, beside them, sum p |v| and the bound
    on a logit's magnitude sum |q| |k| (for tolerances)."""
    out, size, logit = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:2])
    t0 = 0
    for b, n in enumerate(new):
        for h in range(batch.H):
            k, v = (x[b, h, : batch.ctx[b]] for x in batch.rows)
            for i in range(n):
                m = batch.ctx[b] - n + i + 1
                for j in range(h * n_q, (h + 1) * n_q):
                    with np.errstate(invalid="ignore", over="ignore"):
                        s = scale * (k[:m] @ q[t0 + i, j])
                        p = np.exp(s - s.max())
                        p /= p.sum()
                        out[t0 + i, j] = p @ v[:m]
                        size[t0 + i, j] = p @ np.abs(v[:m])
                        logit[t0 + i, j] = scale * np.max(np.abs(k[:m]) @ np.abs(q[t0 + i, j]))
        t0 += n
    return out, size, logit


def _bound(dtype, want, size, logit, tokens, hd, vmax):
    """Derived from the roundings.  16-bit queries: q and k are rounded to
    fp16 (2^-11 each: a logit is off by 2^-10 sum |q| |k| scale), so a weight by
    a factor e^(2 delta) at most; a weight and a value once more by 2^-11 each;
    then the output's own rounding.  fp32: products and sums of hd (logits) and
    of all tokens (output) terms, each by 2^-24, and the exponential's own 2^-22."""
    if dtype == "f32":
        delta = (hd + 4) * 2.0 ** -24 * logit + 2.0 ** -22
        return (2 * np.expm1(2 * delta)[..., None] + (tokens + 8) * 2.0 ** -24) * size + 2.0 ** -24 * np.abs(want)
    delta = 2.0 ** -10 * logit + 2.0 ** -20
    half = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -11
    return (np.expm1(2 * delta)[..., None] + 2.0 ** -10 * (1 + 2.0 ** -6)) * size + half * np.abs(want) + tokens * 2.0 ** -25 * vmax + 2.0 ** -20


def _check(batch, new, n_q, dtype, rng, plan=None, **kw):
    import torch

    T, Hq, hd = int(sum(new)), batch.H * n_q, batch.hd
    # small queries: logits stay of order 1, so that the bounds stay tight
    q = torch.from_numpy((rng.normal(size=(T, Hq, hd)) * 0.5).astype(np.float32)).to(_dt(dtype)).cuda()
    scale = 1.0 / np.sqrt(hd)
    plan = plan or batch.plan(new, n_q, dtype=q.dtype)
    got = batch.attend(q, plan, scale, **kw)
    assert got.shape == q.shape and got.dtype == q.dtype
    want, size, logit = _want(batch, q.double().cpu().numpy(), new, n_q, scale)
    err = np.abs(got.double().cpu().numpy() - want)
    bound = _bound(dtype, want, size, logit, max(batch.ctx), hd, np.max(np.abs(batch.rows[1])))
    assert np.all(err <= bound), float(np.max(err / bound))
    return q, got


_FORMATS = [("a4", "s4"), ("m3", "s8"), ("a8", "a3"), ("s2", "m3_i8"), ("m3_f32", "a2"), ("s3", "m3"), ("s8", "a8")]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("key,value", _FORMATS)
def test_formats(key, value, dtype):
    """Two sequences, a tail page of another format, one row tile and its border."""
    rng = np.random.default_rng(len(key) + len(value))
    print(f"chunk formats {key} {value} {dtype}", flush=True)
    batch = _Batch(rng, [150, 70], 2, 128, 32, key, value)
    _check(batch, [20, 9], 3, dtype, rng, validate=True)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("hd,gs,layout", [(64, (32, 64), "group_major"), (96, (32, 32), "group_major"), (256, (32, 32), "group_major"),
                                          (128, (128, 64), "token_major"), (32, (32, 32), "token_major"), (80, (16, 32), "group_major"),
                                          (30, (32, 32), "group_major"), (40, (24, 8), "group_major"), (200, (64, 40), "group_major"),
                                          (1, (32, 32), "group_major")])
def test_geometries(hd, gs, layout, dtype):
    rng = np.random.default_rng(hd)
    print(f"chunk geometry {hd} {gs} {layout} {dtype}", flush=True)
    batch = _Batch(rng, [131, 300], 1, hd, 64, "a4", "a4", gs, layout=layout)
    _check(batch, [5, 40], 4, dtype, rng)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("P", [1, 10, 16, 24, 48, 100, 256, 300])
def test_page_sizes(P, dtype):
    """Pages that end inside a tile, tiles that end inside a page."""
    rng = np.random.default_rng(P)
    print(f"chunk pages of {P} {dtype}", flush=True)
    batch = _Batch(rng, [201, 77], 1, 64, P, "a4", "s8")
    _check(batch, [33, 77], 2, dtype, rng)


@pytest.mark.parametrize("n_q", [1, 2, 5, 7, 16, 20, 130])
def test_shared_heads(n_q):
    """Row tiles that end inside a token's heads."""
    rng = np.random.default_rng(n_q)
    print(f"chunk n_q {n_q}", flush=True)
    batch = _Batch(rng, [90], 2, 64, 16)
    _check(batch, [30], n_q, "f16", rng)


@pytest.mark.parametrize("new,ctx", [([1], [1]), ([1, 1, 1], [1, 2, 65]), ([64], [64]), ([129], [129]), ([0, 3, 0, 17, 1, 0], [5, 3, 0, 260, 128, 0]),
                                     ([128, 1], [128, 1000]), ([1, 200], [513, 200])])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_lengths(new, ctx, dtype):
    """From one token of one up; sequences that wait; sequences without any."""
    rng = np.random.default_rng(sum(ctx))
    print(f"chunk lengths {new} {ctx} {dtype}", flush=True)
    batch = _Batch(rng, ctx, 2, 64, 64)
    _check(batch, new, 3, dtype, rng)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_split_ranges(hd, dtype):
    """Few rows over a long context, cut into many ranges and joined; the same
    rows whole give the same within the bound, and twice the same bits."""
    import torch

    rng = np.random.default_rng(hd)
    print(f"chunk split {hd} {dtype}", flush=True)
    batch = _Batch(rng, [3100, 700], 1, hd, 64)
    new = [4, 90]
    many = batch.plan(new, 2, target_items=64, dtype=_dt(dtype))
    assert many.n_partials > 8 and many.n_merges >= 2
    q, got = _check(batch, new, 2, dtype, rng, plan=many)
    assert torch.equal(got, batch.attend(q, many, 1.0 / np.sqrt(hd)))
    whole = batch.plan(new, 2, target_items=1, dtype=_dt(dtype))
    assert whole.n_partials == 0
    _check(batch, new, 2, dtype, rng, plan=whole)


def test_mixed_page_formats_in_one_stream():
    """Keys exact in every other page, as a selective precision map keeps them."""
    import torch

    rng = np.random.default_rng(3)
    batch = _Batch(rng, [500], 2, 128, 16, "a4", "s4")
    pool, table = batch.pools[0], batch.host[0]
    for p in range(0, 30, 2):
        table[0, :, p] = pool.allocate(0, 0, 2, tokens=16)
    x = rng.normal(size=(2, 30 * 16, 128)).astype(np.float32)
    t = np.arange(30 * 16)
    pool.encode_rows(torch.from_numpy(x.reshape(-1, 128)).cuda(), np.ascontiguousarray(table[0][:, t // 16]).reshape(-1),
                     np.tile(t % 16, 2).astype(np.int32))
    batch.tables[0] = torch.from_numpy(table).cuda()
    batch.read()
    for dtype in ("f32", "f16"):
        _check(batch, [60], 4, dtype, rng, validate=True)


def test_strided_and_padded_queries():
    """Queries as a view of a projection, out with rows behind the last
    sequence's and unaligned rows: the rest stays as it was."""
    import torch

    rng = np.random.default_rng(4)
    hd, n_q, H = 64, 3, 2
    batch = _Batch(rng, [100, 40], H, hd, 16)
    new = [9, 4]
    plan = batch.plan(new, n_q)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        fused = torch.from_numpy(rng.normal(size=(16, H * n_q + 5, hd)).astype(np.float32)).to(dtype).cuda()
        q = fused[:, 2: 2 + H * n_q]
        want = batch.attend(q[:13].contiguous(), plan, 0.2)
        store = torch.full((16 * (H * n_q * hd + 1) + 1,), 5.0, dtype=dtype, device="cuda")
        out = store[1:].view(16, H * n_q * hd + 1)[:, 1:].view(16, H * n_q, hd)
        assert batch.attend(q, plan, 0.2, out=out) is out
        assert torch.equal(out[:13], want) and torch.all(out[13:] == 5.0)
        assert torch.all(store[1:].view(16, -1)[:, 0] == 5.0) and store[0] == 5.0
        with pytest.raises(ValueError):
            batch.attend(q, plan, 0.2)  # 16 rows, a plan for 13, no out


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("value", ["m3", "m3_f32", "s4"])
def test_values_that_are_not_finite(value, dtype):
    """An infinity or NaN in a new token's value, in a key that a row does not
    see, and in slots behind the last token reaches the rows that see it, in
    its channel, and no others."""
    import torch

    rng = np.random.default_rng(5)
    hd, n = 64, 50
    batch = _Batch(rng, [180], 1, hd, 32, "m3", value, tail=False)
    x = torch.from_numpy(rng.normal(size=(1, hd)).astype(np.float32)).cuda()
    bad = x.clone()
    bad[0, 5], bad[0, 40] = float("inf"), float("nan")
    at = lambda u: ([int(batch.host[1][0, 0, u // 32])], [u % 32])  # noqa: E731
    batch.pools[1].encode_rows(bad, *at(150))  # new token 20 of 50
    batch.pools[1].encode_rows(bad, *at(185))  # behind the last token
    batch.pools[0].encode_rows(bad, [int(batch.host[0][0, 0, 5])], [10])  # the key of token 170
    batch.read()
    q = torch.from_numpy((0.5 * rng.normal(size=(n, 2, hd))).astype(np.float32)).to(_dt(dtype)).cuda()
    plan = batch.plan([n], 2, dtype=q.dtype)
    got = batch.attend(q, plan, 0.125).double().cpu().numpy()
    want, size, logit = _want(batch, q.double().cpu().numpy(), [n], 2, 0.125)
    assert np.isfinite(want[:20]).all() and not np.isfinite(want[20:40]).all() and np.isnan(want[40:]).all()
    assert np.array_equal(np.isfinite(got), np.isfinite(want))
    if value != "s4":  # (a code's infinite scale: s (c - z) is an infinity where s c - s z is NaN)
        assert np.array_equal(np.isnan(got), np.isnan(want))
    fin = np.isfinite(want)
    bound = _bound(dtype, want, size, logit, 180, hd, np.max(np.abs(batch.rows[1][np.isfinite(batch.rows[1])])))
    assert np.all(np.abs(got[fin] - want[fin]) <= bound[fin])


def test_tokens_without_a_page():
    """Page ids that the pools do not hold and pages short of tokens are left
    out, never read; a row that then sees nothing gives zeros."""
    import torch

    from dotcache_amd.chunk import attend_chunk

    rng = np.random.default_rng(6)
    hd, P = 64, 16
    batch = _Batch(rng, [64, 16], 1, hd, P, tail=False)
    for dtype in ("f32", "f16"):
        q = torch.from_numpy(rng.normal(size=(12, 1, hd)).astype(np.float32)).to(_dt(dtype)).cuda()
        plan = batch.plan([10, 2], 1, dtype=q.dtype)
        kt, vt = (t.clone() for t in batch.tables)
        kt[0, 0, 1] = 10 ** 6
        vt[0, 0, 2] = -5
        kt[1, 0, 0] = -1
        batch.pools[0].set_tokens([int(batch.host[0][0, 0, 0])], 7)
        got = attend_chunk(batch.pools[0], kt, batch.pools[1], vt, q, plan, query_scale=0.125).double().cpu().numpy()
        with pytest.raises(ValueError):
            attend_chunk(batch.pools[0], kt, batch.pools[1], vt, q, plan, validate=True)
        batch.pools[0].set_tokens([int(batch.host[0][0, 0, 0])], P)
        keep = np.r_[0:7, 48:64]
        for i in range(10):
            use = keep[keep <= 54 + i]
            k, v = (x[0, 0, use] for x in batch.rows)
            s = 0.125 * (k @ q[i, 0].double().cpu().numpy())
            p = np.exp(s - s.max())
            want = p @ v / p.sum()
            # (fp16 operands: logits of order 4 off by 2^-10 of their terms' sum, about 2^-6)
            assert np.max(np.abs(got[i, 0] - want)) <= (2.0 ** -5 if dtype == "f16" else 2.0 ** -16) * np.max(np.abs(v))
        assert np.all(got[10:] == 0)


def test_two_streams_and_a_graph():
    """Calls at once on two streams, each with a workspace of its own, and
    replays of a captured call with eager work between."""
    import torch

    rng = np.random.default_rng(7)
    batch = _Batch(rng, [2000, 900], 2, 128, 64)
    new = [6, 70]
    plan = batch.plan(new, 4, target_items=200)
    assert plan.n_partials > 0
    qs = [torch.randn(76, 8, 128, device="cuda").half() for _ in range(2)]
    want = [batch.attend(q, plan, 0.09) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(batch.attend(qs[i], plan, 0.09))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])
    q = qs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = batch.attend(q, plan, 0.09)
    for i in range(4):
        q.copy_(qs[i % 2])
        graph.replay()
        held = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(held, want[i % 2]) and torch.equal(batch.attend(qs[1], plan, 0.09), want[1])


def test_long_offsets():
    """A pool whose pages lie past 2^32 bytes, and a table wider than the context."""
    import torch

    rng = np.random.default_rng(8)
    batch = _Batch(rng, [300], 1, 128, 64, "m3", "m3", spare=3)
    want_rows = [x.copy() for x in batch.rows]
    from dotcache_amd.page_pool import DevicePagePool

    far = []
    for pool, table in zip(batch.pools, batch.host):
        big = DevicePagePool(pool.geometry, reserve_bytes=(1 << 32) + (1 << 24), reserve_pages=1 << 19)
        big._next_block = (1 << 24) - 40  # blobs around 4 GiB
        ids = big.allocate(0, 0, table.size, tokens=64).reshape(table.shape).astype(np.int32)
        big.set_tokens(ids[0, :, 4], 300 - 256)
        far.append((big, ids))
    for i, (big, ids) in enumerate(far):
        x = torch.from_numpy(want_rows[i][0, 0].astype(np.float32)).cuda()
        t = np.arange(x.shape[0])
        big.encode_rows(x, ids[0, 0, t // 64], (t % 64).astype(np.int32))
        batch.pools[i], batch.host[i], batch.tables[i] = big, ids, torch.from_numpy(ids).cuda()
    batch.read()
    assert all(np.array_equal(a, b) for a, b in zip(batch.rows, want_rows))
    _check(batch, [33], 2, "f16", rng)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("n", [5, 50])
@pytest.mark.parametrize("value", ["m3", "m3_f32"])
def test_an_infinity_where_a_range_begins(value, n, dtype):
    """A range's first tile has no maximum to rescale from: an infinity there
    stays one for the rows that see it, with few rows and many."""
    import torch

    rng = np.random.default_rng(n)
    hd, ctx = 64, 300
    print(f"chunk infinity {value} {n} {dtype}", flush=True)
    batch = _Batch(rng, [ctx], 1, hd, 32, "m3", value, tail=False)
    bad = torch.from_numpy(rng.normal(size=(1, hd)).astype(np.float32)).cuda()
    bad[0, 7] = float("inf")
    u = ctx - n + 2 if n < 44 else 258  # in the last range of 128, seen by some of the rows
    batch.pools[1].encode_rows(bad, [int(batch.host[1][0, 0, u // 32])], [u % 32])
    batch.read()
    q = torch.from_numpy((0.5 * rng.normal(size=(n, 2, hd))).astype(np.float32)).to(_dt(dtype)).cuda()
    plan = batch.plan([n], 2, dtype=q.dtype, target_items=64)
    assert plan.n_partials > 0
    got = batch.attend(q, plan, 0.125).double().cpu().numpy()
    first = u - (ctx - n)  # the first row that sees it
    assert np.isposinf(got[first:, :, 7]).all() and np.isfinite(got[:first]).all()
    assert np.isfinite(np.delete(got, 7, axis=2)).all()
