"""Norms with rotation, the append that rotates on its way into the pages, and
dense reads of pages, against fp64 numpy and the oracle's encoder: head_dims
off the 8-channel lanes, partial and interleaved rotations, strided views,
every page format, tokens without a page, positions outside the table, and
captured replays."""
import numpy as np
import pytest

from oracle import dotcache_oracle as O

pytestmark = pytest.mark.gpu


def _dt(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


# half a step of the output type, and of fp32 for the few operations before it:
# y = x r w (r a square root of a sum of squares, all in fp32: each operation
# off by at most 2^-24, the sum of hd squares by hd 2^-24, halved by the root)
# and two products and a sum per pair, whose terms are at most |y| + |y'|
_HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def _rotate64(x, weight, positions, table, rd, interleaved, eps):
    """fp64 rows and, per element, the sum of the magnitudes of its terms."""
    y = x.astype(np.float64)
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * weight.astype(np.float64)
    out, size = y.copy(), np.abs(y)
    if rd:
        cos, sin = (t[:, None, :].astype(np.float64) for t in np.split(table[positions], 2, axis=-1))
        a, b = (slice(0, rd, 2), slice(1, rd, 2)) if interleaved else (slice(0, rd // 2), slice(rd // 2, rd))
        out[..., a] = y[..., a] * cos - y[..., b] * sin
        out[..., b] = y[..., b] * cos + y[..., a] * sin
        size[..., a] = np.abs(y[..., a] * cos) + np.abs(y[..., b] * sin)
        size[..., b] = np.abs(y[..., b] * cos) + np.abs(y[..., a] * sin)
    return out, size


def _close(got, want, size, dtype, hd):
    bound = _HALF[dtype] * np.abs(want) + (hd / 2 + 8) * 2.0 ** -24 * size + 2.0 ** -24  # (fp16's subnormal step)
    err = np.abs(got.float().cpu().numpy().astype(np.float64) - want)
    assert np.all(err <= bound), float((err / bound).max())


# (head_dim, rotary_dim, interleaved): whole rows on lanes; rotations of a part;
# pairs that start inside a lane's 8 channels; head_dims that are no multiple of 8;
# rows longer than a wavefront's lanes
_SHAPES = [(128, 128, False), (64, 64, True), (256, 64, False), (96, 48, False), (96, 40, True), (80, 20, False),
           (40, 36, True), (30, 30, False), (7, 2, True), (576, 64, False), (128, 0, False),
           (72, 32, False), (88, 24, True), (24, 8, True), (512, 512, False)]  # (lanes with one chunk of eight; 32 lanes a row)


@pytest.mark.parametrize("hd,rd,interleaved", _SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_norm_rotate(hd, rd, interleaved, dtype):
    import torch

    from dotcache_amd.rotary import RotaryTable, norm_rotate

    rng = np.random.default_rng(hd * 7 + rd)
    for T, norm in ((1, True), (37, False), (37, True)):
        print(f"norm_rotate hd {hd} rd {rd} {interleaved} {dtype} T {T} norm {norm}", flush=True)
        fused = torch.from_numpy(rng.normal(size=(T, 7, hd)).astype(np.float32)).to(_dt(dtype)).cuda()
        q, k = fused[:, :5], fused[:, 5:7]  # views of one projection
        rotary = RotaryTable(hd, 500, rotary_dim=rd, interleaved=interleaved, base=500.0) if rd else None
        pos = rng.integers(0, 500, T)
        qw = rng.normal(size=(hd,)).astype(np.float32) if norm else None
        kw = rng.normal(size=(2, hd)).astype(np.float32) if norm else None  # one weight per head
        got = norm_rotate(q, k, torch.from_numpy(pos).cuda(), rotary,
                          q_weight=None if qw is None else torch.from_numpy(qw).cuda(),
                          k_weight=None if kw is None else torch.from_numpy(kw).cuda(), eps=1e-5)
        table = rotary.table.cpu().numpy() if rd else None
        for x, y, w in ((q, got[0], qw), (k, got[1], kw)):
            want, size = _rotate64(x.float().cpu().numpy(), w, pos, table, rd, interleaved, np.float64(np.float32(1e-5)))
            assert y.dtype == x.dtype and y.shape == x.shape
            _close(y, want, size, dtype, hd)


def test_table_holds_far_angles():
    """cos and sin of position 10^6: fp32 angles would be off by up to 0.03."""
    from dotcache_amd.rotary import RotaryTable

    t = RotaryTable(8, 1000001, rotary_dim=4, inv_freq=[1.0, 0.37]).table[1000000].cpu().numpy().astype(np.float64)
    a = 1e6 * np.array([1.0, 0.37])
    assert np.all(np.abs(t - np.concatenate([np.cos(a), np.sin(a)])) <= 2.0 ** -24)


@pytest.mark.parametrize("hd,rd", [(128, 128), (30, 30)])
def test_norm_rotate_places(hd, rd):
    """In place, into fp32 rows, unaligned rows, one side alone, no tokens, and
    positions outside the table."""
    import torch

    from dotcache_amd.rotary import RotaryTable, norm_rotate

    rng = np.random.default_rng(5)
    rotary = RotaryTable(hd, 100, rotary_dim=rd)
    x = torch.from_numpy(rng.normal(size=(11, 3, hd)).astype(np.float32)).bfloat16().cuda()
    pos = torch.arange(11, device="cuda", dtype=torch.int32)
    want = norm_rotate(x, None, pos, rotary)[0]
    assert norm_rotate(x, None, pos, rotary)[1] is None
    assert torch.equal(norm_rotate(None, x, pos, rotary)[1], want)
    wide = torch.empty(11, 3, hd, device="cuda")
    norm_rotate(x, None, pos, rotary, out=(wide, None))
    assert torch.equal(wide.bfloat16(), want)
    store = torch.zeros(11 * 3 * hd + 1, device="cuda", dtype=torch.bfloat16)
    y = store[1:].view(11, 3, hd)  # rows off 16 bytes
    y.copy_(x)
    assert norm_rotate(y, None, pos, rotary, out=(y, None))[0] is y
    assert torch.equal(y, want) and store[0] == 0
    assert norm_rotate(x[:0], x[:0], pos[:0], rotary)[0].shape == (0, 3, hd)
    bad = pos.clone()
    bad[[2, 7]] = torch.tensor([100, -1], device="cuda", dtype=torch.int32)
    got = norm_rotate(x, None, bad, rotary)[0]
    keep = [i for i in range(11) if i not in (2, 7)]
    assert torch.isnan(got[[2, 7]]).all() and torch.equal(got[keep], want[keep])
    far = torch.tensor([2 ** 40] * 11, device="cuda")  # (not a position once cut to 32 bits)
    assert torch.isnan(norm_rotate(x, None, far, rotary)[0]).all()


_FORMATS = [("a4", "s4"), ("m3", "s8"), ("a8", "a3"), ("s2", "m3_i8"), ("m3_f32", "a2"), ("s3", "m3")]


def _form(name):
    from dotcache_amd.page_pool import page_format_of

    if name.startswith("m3"):
        return page_format_of("M3", "affine", 4, {"m3": "float16", "m3_i8": "int8", "m3_f32": "float32"}[name])
    return page_format_of("M0", "affine" if name[0] == "a" else "symmetric", int(name[1:]))


def _oracle_page(rows, name, hd, gs, kind):
    if name.startswith("m3"):
        return O.encode_page(rows, head_dim=hd, group_size=gs, bits=4, kind=kind, mode="M3",
                             escape_dtype={"m3": "float16", "m3_i8": "int8", "m3_f32": "float32"}[name])
    return O.encode_page(rows, head_dim=hd, group_size=gs, bits=int(name[1:]), kind=kind, mode="M0",
                         scheme="affine" if name[0] == "a" else "symmetric")


def _same(page, want, slots):
    """The page's slots hold the oracle page's rows, bit for bit."""
    for field in ("payload", "scales", "bias", "escape_payload", "escape_scales"):
        a, b = getattr(page, field), getattr(want, field)
        assert (a is None) == (b is None), field
        if a is not None:
            a = a[:, slots] if field == "payload" else a[slots]
            assert np.array_equal(np.ascontiguousarray(a).view(np.uint8), np.ascontiguousarray(b).view(np.uint8)), field


def _dense(name, page):
    """fp32 rows of an oracle page, from its fields alone."""
    if page.payload is None:
        x = page.escape_payload.astype(np.float32)
        return x * page.escape_scales.astype(np.float32)[:, None] if page.escape_scales is not None else x
    h = page.header
    G, T, W = page.payload.shape
    bits, gs = h.bits, h.group_size
    stream = np.unpackbits(page.payload.view(np.uint8).reshape(G, T, W * 4), axis=-1, bitorder="little")
    codes = (stream[..., : gs * bits].reshape(G, T, gs, bits) * (1 << np.arange(bits))).sum(-1).astype(np.float32)
    s = page.scales.astype(np.float32).T[..., None]
    if name[0] == "a":
        x = codes * s + page.bias.astype(np.float32).T[..., None]
    else:
        x = (codes - ((1 << (bits - 1)) - 1)) * s
    return x.transpose(1, 0, 2).reshape(T, G * gs)[:, : h.head_dim]


@pytest.mark.parametrize("hd,gs,rd,interleaved,norm", [(128, 32, 128, False, True), (96, 32, 48, True, False),
                                                        (64, 64, 64, False, False), (256, 32, 128, False, True),
                                                        (30, 32, 20, False, True), (80, 16, 40, False, False)])
@pytest.mark.parametrize("key,value", _FORMATS)
def test_append_rotary_pages(hd, gs, rd, interleaved, norm, key, value):
    """Two sequences' tokens across page borders: the pages hold what encoding
    the fp64 formula's rows gives, and read back as the values they stand for."""
    import torch

    from dotcache_amd.page_pool import DevicePagePool, PoolGeometry
    from dotcache_amd.rotary import RotaryTable, norm_rotate

    P, H, Hq, B, n, first = 16, 2, 3, 2, 21, (13, 0)
    print(f"append_rotary hd {hd} gs {gs} rd {rd} {key} {value}", flush=True)
    rng = np.random.default_rng(hd + rd)
    fused = torch.from_numpy(rng.normal(size=(B * n, Hq + 2 * H, hd)).astype(np.float32)).bfloat16().cuda()
    q, k, v = fused[:, :Hq], fused[:, Hq: Hq + H], fused[:, Hq + H:]
    pools = [DevicePagePool(PoolGeometry(hd, gs, P), reserve_bytes=1 << 18, reserve_pages=32) for _ in range(2)]
    forms = [_form(key), _form(value)]
    W = 3
    ids = np.stack([rng.permutation(p.allocate(*f, B * H * W, tokens=P)).reshape(B, H, W) for p, f in zip(pools, forms)])
    tables = torch.from_numpy(ids.astype(np.int32)).cuda()
    token = np.concatenate([f + np.arange(n) for f in first])
    row = np.repeat(np.arange(B), n)
    pos = np.concatenate([100 + np.arange(n), 4000 + np.arange(n)])
    rotary = RotaryTable(hd, 5000, rotary_dim=rd, interleaved=interleaved)
    w = (1 + 0.1 * rng.normal(size=(2, hd))).astype(np.float32) if norm else (None, None)
    qw, kw = (None if x is None else torch.from_numpy(x).cuda() for x in w)
    keep_rows = torch.full((2, B * H * W * P, hd), 7.0, device="cuda")
    keep_row = np.where(token % 2 == 0, row * H * W * P + token, -1)
    out = pools[0].append_rotary_with(pools[1], q, k, v, pos, rotary, tables, row, token, q_weight=qw, k_weight=kw,
                                      keep=(keep_rows[0], keep_rows[1], keep_row, W * P))
    assert torch.equal(out, norm_rotate(q, None, pos, rotary, q_weight=qw)[0])
    table = rotary.table.cpu().numpy()
    k64, _ = _rotate64(k.float().cpu().numpy(), w[1], pos, table, rd, interleaved, np.float64(np.float32(1e-6)))
    rows = (k64.astype(np.float32), v.float().cpu().numpy())
    back = pools[0].read_tokens_with(pools[1], tables, row, token)
    kept = keep_rows.cpu().numpy()
    for i, (name, kind) in enumerate(((key, "K"), (value, "V"))):
        for b in range(B):
            for h in range(H):
                for p in range(W):
                    at = np.flatnonzero((row == b) & (token // P == p))
                    if at.size == 0:
                        continue
                    want = _oracle_page(rows[i][at, h], name, hd, gs, kind)
                    _same(pools[i].download_page(ids[i, b, h, p], kind=kind), want, token[at] % P)
                    assert np.array_equal(back[i][torch.from_numpy(at).cuda(), h].cpu().numpy(), _dense(name, want))
                    for a in at[keep_row[at] >= 0]:
                        assert np.array_equal(kept[i, keep_row[a] + h * W * P], rows[i][a, h])
    assert np.sum(np.any(kept != 7.0, axis=-1)) == 2 * H * np.sum(keep_row >= 0)
    for dtype in (torch.float16, torch.bfloat16):
        for x, y in zip(pools[0].read_tokens_with(pools[1], tables, row, token, dtype=dtype), back):
            assert torch.equal(x, y.to(dtype))


@pytest.mark.parametrize("hd", [128, 30])
def test_tokens_without_a_page_are_left_out(hd):
    """Padding tokens, rows and pages outside the table, page ids the pool does
    not hold and positions outside the rotation's table: every page byte of the
    others' slots stays, the queries are made all the same, reads give zeros."""
    import torch

    from dotcache_amd.page_pool import DevicePagePool, PoolGeometry
    from dotcache_amd.rotary import RotaryTable

    P, H, T = 16, 2, 8
    rng = np.random.default_rng(1)
    pools = [DevicePagePool(PoolGeometry(hd, 32, P), reserve_bytes=1 << 16, reserve_pages=16) for _ in range(2)]
    ids = np.stack([p.allocate(1, 4, 4, tokens=P).reshape(1, H, 2) for p in pools])
    ids[:, 0, :, 1] = (-1, 999)  # head 0's second page: no page; head 1's: outside the pool
    tables = torch.from_numpy(ids.astype(np.int32)).cuda()
    x = torch.from_numpy(rng.normal(size=(T, 3 * H, hd)).astype(np.float32)).cuda()
    rotary = RotaryTable(hd, 10)
    row = torch.tensor([0, 0, 1, -1, 0, 0, 0, 0], device="cuda", dtype=torch.int32)
    token = torch.tensor([3, -1, 4, 5, P + 2, 2 * P, 2 ** 31 - 1, 6], device="cuda", dtype=torch.int32)
    pos = torch.tensor([1, 2, 3, 4, 5, 6, 7, 10], device="cuda", dtype=torch.int32)
    before = [p.arena.clone() for p in pools]
    for p in pools:
        p.arena.fill_(0xAB)
    q = pools[0].append_rotary_with(pools[1], x[:, :H], x[:, H: 2 * H], x[:, 2 * H:], pos, rotary, tables, row, token)
    assert torch.isfinite(q[:7]).all() and torch.isnan(q[7]).all()
    written = [(p.arena != 0xAB).sum().item() for p in pools]
    alone = []
    for p in pools:  # token 0 alone
        p.arena.fill_(0xAB)
    pools[0].append_rotary_with(pools[1], None, x[:1, H: 2 * H], x[:1, 2 * H:], pos[:1], rotary, tables, row[:1], token[:1])
    alone = [(p.arena != 0xAB).sum().item() for p in pools]
    assert written == alone
    got = pools[0].read_tokens_with(pools[1], tables, row, token)
    for i, y in enumerate(got):
        assert torch.all(y[1:7] == 0) and torch.any(y[0] != 0)
    del before


def test_append_in_a_graph_and_on_another_stream():
    """A captured append replays on new rows, with eager work between; another
    stream's append and read are ordered on that stream."""
    import torch

    from dotcache_amd.page_pool import DevicePagePool, PoolGeometry
    from dotcache_amd.rotary import RotaryTable

    hd, P, H, T = 128, 16, 2, 5
    pools = [DevicePagePool(PoolGeometry(hd, 32, P), reserve_bytes=1 << 18, reserve_pages=32) for _ in range(2)]
    ids = np.stack([p.allocate(1, 4, T * H, tokens=P).reshape(T, H, 1) for p in pools])
    tables = torch.from_numpy(ids.astype(np.int32)).cuda()
    row = torch.arange(T, device="cuda", dtype=torch.int32)
    token = torch.full((T,), 3, device="cuda", dtype=torch.int32)
    pos = torch.arange(T, device="cuda", dtype=torch.int32)
    rotary = RotaryTable(hd, 64)
    x = torch.randn(T, 3 * H, hd, device="cuda").bfloat16()
    w = torch.ones(hd, device="cuda")

    def step():
        q = pools[0].append_rotary_with(pools[1], x[:, :H], x[:, H: 2 * H], x[:, 2 * H:], pos, rotary, tables, row, token,
                                        q_weight=w, k_weight=w)
        return (q, *pools[0].read_tokens_with(pools[1], tables, row, token, dtype=torch.bfloat16))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        x.copy_(torch.randn(T, 3 * H, hd, device="cuda") * (i + 1))
        graph.replay()
        got = [y.clone() for y in held]
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
    x.copy_(torch.randn(T, 3 * H, hd, device="cuda"))
    want = step()
    for p in pools:
        p.arena.zero_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [128, 96])
def test_large_calls_are_small_calls_side_by_side(hd, dtype):
    """Calls whose rows the caches would not hold store past them, and lanes take
    several heads: the same bits as the same rows in small calls."""
    import torch

    from dotcache_amd.page_pool import DevicePagePool, PoolGeometry
    from dotcache_amd.rotary import RotaryTable, norm_rotate

    dt = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    T, heads, small = 24001, 7, 900
    torch.manual_seed(hd)
    x = torch.randn(T, heads, hd, device="cuda").to(dt)
    w = torch.rand(hd, device="cuda") + 0.5
    rotary = RotaryTable(hd, 4096, rotary_dim=hd // 3 // 32 * 32 + 32)
    pos = torch.randint(0, 4096, (T,), dtype=torch.int32, device="cuda")
    y, _ = norm_rotate(x, None, pos, rotary, q_weight=w)
    for a in range(0, T, small):
        z, _ = norm_rotate(x[a: a + small], None, pos[a: a + small], rotary, q_weight=w)
        assert torch.equal(z, y[a: a + small])
    pools = [DevicePagePool(PoolGeometry(hd, 32, 64), reserve_bytes=1 << 20, reserve_pages=64) for _ in range(2)]
    tables = []
    for p, form in zip(pools, (_form("a4"), _form("s3"))):
        ids = p.allocate(*form, 2 * 5 * 3, tokens=64)
        p.encode_rows(torch.randn(30 * 64, hd, device="cuda"), np.repeat(ids, 64), np.tile(np.arange(64), 30))
        tables.append(torch.from_numpy(np.asarray(ids, dtype=np.int32).reshape(2, 5, 3)).cuda())
    tables = torch.stack(tables).contiguous()
    row = torch.randint(-1, 3, (T,), dtype=torch.int32, device="cuda")  # (some tokens without a page)
    token = torch.randint(0, 3 * 64, (T,), dtype=torch.int32, device="cuda")
    k, v = pools[0].read_tokens_with(pools[1], tables, row, token, dtype=dt)
    for a in range(0, T, small):
        kk, vv = pools[0].read_tokens_with(pools[1], tables, row[a: a + small], token[a: a + small], dtype=dt)
        assert torch.equal(kk, k[a: a + small]) and torch.equal(vv, v[a: a + small])
