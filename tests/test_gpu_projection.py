"""Products with grouped 4-bit weights: exactly, where inputs, scales and biases
are whole numbers and powers of two (every sum is then exact in fp32, so an
output is the fp64 product rounded once), and within derived bounds elsewhere."""
import numpy as np
import pytest

from tests.test_gpu_chunk import _dt
from tests.test_projection_host import make

pytestmark = pytest.mark.gpu

HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def exact_case(M, K, N, gs, affine, dtype, seed=0):
    """Rows, weight and the outputs, rounded once: |x| <= 3, scales 1/2 .. 2, biases
    multiples of 1/2 up to 8: sums of K products below 3 * 40 * K, in steps of 1/2."""
    import torch

    from dotcache_amd.projection import GroupedWeight

    assert 3 * 40 * K * 2 < 2 ** 24
    r = np.random.default_rng(seed)
    G = -(-K // gs)
    codes = torch.from_numpy(r.integers(0, 16 if affine else 15, size=(N, K)).astype(np.int16)).cuda()
    scales = torch.from_numpy(2.0 ** r.integers(-1, 2, size=(N, G))).half().cuda()
    biases = torch.from_numpy(r.integers(-16, 17, size=(N, G)) / 2.0).half().cuda() if affine else None
    x = torch.from_numpy(r.integers(-3, 4, size=(M, K)).astype(np.float32)).to(_dt(dtype)).cuda()
    g = torch.arange(K, device="cuda") // gs
    dense = codes.double() * scales.double()[:, g] + biases.double()[:, g] if affine else (codes.double() - 7) * scales.double()[:, g]
    want = x.double() @ dense.t().contiguous()
    return x, GroupedWeight.from_codes(codes, scales, biases, group_size=gs), want.to(_dt(dtype)), dense


SIZES = [(1, 128, 16), (1, 1, 1), (20, 7, 300), (3, 8, 40), (70, 15, 33), (2, 31, 5), (3, 160, 17), (16, 128, 33), (17, 257, 48), (5, 1000, 777), (33, 1024, 64), (1, 3584, 129), (64, 640, 130),
         (65, 512, 100), (130, 96, 257), (128, 64, 256), (300, 448, 272), (513, 130, 16), (257, 2048, 144)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("gs,affine", [(32, True), (64, True), (128, True), (32, False), (64, False), (128, False)])
def test_exact(gs, affine, dtype):
    import torch

    from dotcache_amd.projection import project

    for i, (M, K, N) in enumerate(SIZES):
        print(f"project {M} {K} {N} {gs} {affine} {dtype}", flush=True)
        x, w, want, _ = exact_case(M, K, N, gs, affine, dtype, i)
        got = project(x, w)
        assert got.dtype == x.dtype and torch.equal(got, want), (M, K, N)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M", [1, 7, 40, 200])
def test_rounded(M, dtype):
    """Any values: whole-number operands are exact, so an output is off by its
    sums' fp32 roundings (2^-23 for each of a group's terms and of the groups,
    of at most (31 scale + |offset|) |x|), and by its own."""
    import torch

    from dotcache_amd.projection import GroupedWeight, project

    K, N, gs = 700, 100, 64
    codes, scales, biases, dense = make(N, K, gs, True, M, "cuda")
    w = GroupedWeight.from_codes(codes, scales, biases, group_size=gs)
    r = np.random.default_rng(M)
    x = torch.from_numpy((r.normal(size=(M, K)) * np.exp(r.normal(size=(1, K)))).astype(np.float32)).to(_dt(dtype)).cuda()
    got, xs = project(x, w).double().cpu().numpy(), x.double().cpu().numpy()
    want = xs @ dense.T
    g = np.arange(K) // gs
    s, b = (t.double().cpu().numpy()[:, g] for t in (scales, biases))
    size = np.abs(xs) @ (31 * s + np.abs(b - 16 * s)).T
    # (16-bit rows of large calls: a weight is rounded to fp16 once)
    few = 0.0 if M <= 64 or dtype == "f32" else 2.0 ** -11 * (np.abs(xs) @ np.abs(dense).T)
    bound = (gs + -(-K // gs) + 16) * 2.0 ** -23 * size + few + HALF[dtype] * np.abs(want) + 2.0 ** -20
    assert np.all(np.abs(got - want) <= bound), float(np.max(np.abs(got - want) / bound))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M", [1, 9, 70, 300])
def test_strides_and_rows_apart(M, dtype):
    """Rows that are views, at odd addresses too, into an output between other
    columns and rows; leading dimensions; one row of any."""
    import torch

    from dotcache_amd.projection import project

    x, w, want, _ = exact_case(M, 200, 50, 32, True, dtype)
    for off, width in ((0, 200), (3, 211), (8, 224)):
        wide = torch.full((M + 2, width + off), float("nan"), dtype=x.dtype, device="cuda")
        rows = wide[1: 1 + M, off: off + 200]
        rows.copy_(x)
        out = torch.full((M + 2, 57), 5.0, dtype=x.dtype, device="cuda")
        got = project(rows, w, out=out[1: 1 + M, 4:54])
        assert got.data_ptr() == out[1:, 4:].data_ptr() and torch.equal(got, want)
        assert bool((out[0] == 5).all() and (out[-1] == 5).all() and (out[:, :4] == 5).all() and (out[:, 54:] == 5).all())
    assert torch.equal(project(x[:, None, :], w), want[:, None, :]) and torch.equal(project(x[0], w), want[0])
    assert torch.equal(project(x[:1].expand(M, 200), w), want[:1].expand(M, 50))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M", [3, 70, 300])
def test_values_that_are_not_finite_stay_in_their_rows(M, dtype):
    import torch

    from dotcache_amd.projection import project

    x, w, want, _ = exact_case(M, 300, 40, 64, True, dtype)
    x[1, 7], x[M - 1, 299] = float("inf"), float("nan")
    got = project(x, w)
    rows = [i for i in range(M) if i not in (1, M - 1)]
    assert torch.equal(got[rows], want[rows]) and not torch.isfinite(got[[1, M - 1]]).any()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("M", [2, 200])
def test_large_and_small_values(M, dtype):
    """Rows over the whole range of their type: beside a row's largest value,
    small ones count as far as fp32 sums keep them, and alone in full."""
    import torch

    from dotcache_amd.projection import project

    x, w, _, dense = exact_case(M, 160, 24, 32, True, dtype)
    top = 2.0 ** 10 if dtype == "f16" else 2.0 ** 100
    for f in (top, 1.0 / top):
        y = x * f
        got = project(y, w).double()
        want = y.double() @ dense.t().contiguous()
        assert torch.equal(got, want.to(y.dtype).double()), f
    if dtype == "bf16":
        y = x.clone()
        y[:, :32] *= 2.0 ** 60
        got, want = project(y, w).double(), y.double() @ dense.t().contiguous()
        size = y.double().abs() @ (dense.abs().t().contiguous() + 40)
        assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -14 * size).all())


def test_quantize_is_the_page_encoder():
    """Levels of a matrix's groups as the framework's pages hold them."""
    import torch

    from dotcache_amd.page_pool import DevicePagePool, PoolGeometry, page_format_of
    from dotcache_amd.projection import GroupedWeight

    for scheme in ("affine", "symmetric"):
        for N, K, gs, dtype in ((40, 256, 32, "f32"), (17, 200, 64, "bf16"), (300, 128, 128, "f16")):
            w = torch.from_numpy(np.random.default_rng(N).normal(size=(N, K)).astype(np.float32)).to(_dt(dtype)).cuda()
            pool = DevicePagePool(PoolGeometry(K, gs, N), reserve_bytes=1 << 16, reserve_pages=16)
            pid = pool.allocate(*page_format_of("M0", scheme, 4), 1, tokens=N)
            pool.encode_rows(w, np.full(N, pid[0], dtype=np.int32), np.arange(N, dtype=np.int32))
            table = torch.from_numpy(pid.reshape(1, 1, 1)).cuda()
            rows, _ = pool.read_tokens_with(pool, torch.stack([table, table]), np.zeros(N, dtype=np.int32), np.arange(N, dtype=np.int32))
            assert torch.equal(GroupedWeight.quantize(w, group_size=gs, scheme=scheme).dense(), rows[:, 0])


def test_replays_and_streams():
    import torch

    from dotcache_amd.projection import project

    cases = [exact_case(M, 384, 80, 64, True, d, M) for M, d in ((1, "bf16"), (40, "f16"), (200, "bf16"), (5, "f32"))]
    side = torch.cuda.Stream()
    for x, w, want, dense in cases:
        assert torch.equal(project(x, w), want)
        out, held = torch.zeros_like(want), x.clone()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            project(held, w, out=out)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            project(held, w, out=out)
        for f in (2.0, 0.5, 1.0, -1.0):
            held.copy_(x * f)
            graph.replay()
            assert torch.equal(out, (x.double() * f @ dense.t().contiguous()).to(out.dtype))
            out.zero_()
            torch.cuda.synchronize()


def test_many_rows():
    """More rows than a launch has blocks in its second dimension."""
    import torch

    from dotcache_amd.projection import project

    x, w, want, _ = exact_case(33, 32, 8, 32, False, "f32")
    many = x.repeat(40000, 1)[: 16 * 65535 + 40]
    got = project(many, w)
    assert torch.equal(got, want.repeat(40000, 1)[: many.shape[0]])


def test_a_layer_of_four_bit_weights_and_pages():
    """One attention layer as a model serves it: queries, keys and values from
    one product, normed, rotated and appended, attended with a window and a cap,
    and the product behind it, for a prompt's chunks and single tokens, against
    fp64 on the same levels."""
    import torch

    from dotcache_amd.chunk import ChunkMask
    from dotcache_amd.config import DotCacheConfig
    from dotcache_amd.kv_cache import DevicePagedKVCache
    from dotcache_amd.projection import GroupedWeight, project
    from dotcache_amd.rotary import RotaryTable, norm_rotate

    Hq, H, hd, hidden, B = 4, 2, 64, 192, 2
    rng = np.random.default_rng(1)
    put = lambda *s: torch.from_numpy(rng.normal(size=s).astype(np.float32)).cuda()  # noqa: E731
    w_in = GroupedWeight.quantize(put((Hq + 2 * H) * hd, hidden) / hidden ** 0.5, group_size=64)
    w_out = GroupedWeight.quantize(put(hidden, Hq * hd) / (Hq * hd) ** 0.5, group_size=32, scheme="symmetric")
    cache = DevicePagedKVCache(DotCacheConfig(head_dim=hd, group_size=32, bits_k=4, bits_v=4, tokens_per_page=16), num_hidden_layers=1,
                               num_attention_heads=Hq, num_key_value_heads=H, batch_size=B)
    rotary = RotaryTable(hd, 256)
    norm, mask, cap, scale = put(hd) * 0.1 + 1, ChunkMask(window=24, sinks=3), 6.0, hd ** -0.5
    at = 0
    for n in (40, 1, 1, 7, 1):
        x = put(B, n, hidden).bfloat16()
        qkv = project(x, w_in).view(B, n, Hq + 2 * H, hd)
        q, k, v = (t.transpose(1, 2) for t in qkv.split([Hq, H, H], dim=2))
        q = cache.append_rotated(0, q, k, v, at, rotary, q_weight=norm, k_weight=norm)
        at += n
        mixed = cache.attend_chunk(0, q, query_scale=scale, mask=mask, cap=cap)
        got = project(mixed.transpose(1, 2).reshape(B, n, Hq * hd), w_out).double().cpu()
        # fp64 from the rows that each step had
        want_qkv = x.double() @ w_in.dense().double().t().contiguous()
        assert bool(((qkv.reshape(B, n, -1).double() - want_qkv).abs() <= 2.0 ** -8 * want_qkv.abs() + 1e-4).all())
        keys, values = (t.double().cpu() for t in cache.read_layer(0))
        i, u = torch.arange(at - n, at)[:, None], torch.arange(at)[None, :]
        sees = (u <= i) & ((u > i - 24) | (u < 3))
        qd = q.double().cpu()
        s = cap * torch.tanh(scale * (qd @ keys.repeat_interleave(Hq // H, 1).transpose(-1, -2)) / cap)
        o = torch.softmax(s.masked_fill(~sees, -np.inf), -1) @ values.repeat_interleave(Hq // H, 1)
        # bf16 outputs, fp16 operands: 2^-8 of the output and 2^-10 of a logit's terms (|q| |k| < 60 at most here)
        assert bool(((mixed.double().cpu() - o).abs() <= 2.0 ** -8 * o.abs() + 0.03).all())
        want = mixed.transpose(1, 2).reshape(B, n, -1).double().cpu() @ w_out.dense().double().cpu().t()
        assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + 1e-4).all())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("gs,affine", [(32, True), (64, True), (128, True), (32, False), (64, False), (128, False)])
def test_tiles(gs, affine, dtype):
    """Calls of many rows at both tile heights: outputs that fill no tile, rows
    at odd addresses and strides, inputs that fill no tile, a workspace of one's own."""
    import torch

    from dotcache_amd.projection import project, workspace_bytes

    for M, K, N in ((1030, 256, 1100), (1152, 200, 2688), (2000, 384, 640), (1100, 1024, 1031)):
        print(f"project tiles {M} {K} {N} {gs} {affine} {dtype}", flush=True)
        x, w, want, _ = exact_case(M, K, N, gs, affine, dtype, M)
        need = workspace_bytes(w, x.dtype, M)
        assert (need > 0) == (dtype == "bf16" or K % 128 != 0)
        assert torch.equal(project(x, w), want)
        wide = torch.full((M + 1, K + 11), float("nan"), dtype=x.dtype, device="cuda")
        rows = wide[1:, 3: 3 + K]
        rows.copy_(x)
        out = torch.full((M, N + 5), 5.0, dtype=x.dtype, device="cuda")
        work = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
        got = project(rows, w, out=out[:, 3: 3 + N], workspace=work)
        assert torch.equal(got, want) and bool((out[:, :3] == 5).all() and (out[:, 3 + N:] == 5).all())
        if need:
            for bad in (work[:-1], torch.empty(need + 8, dtype=torch.uint8, device="cuda")[8:], torch.empty(need, dtype=torch.uint8)):
                with pytest.raises(ValueError):
                    project(x, w, workspace=bad)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_tiles_round_weights_once(dtype):
    """Any values, many rows: a weight is rounded to fp16 (2^-11), its products summed in
    fp32 (2^-23 for each term); rows apart by 2^60 in size, and rows of zeros."""
    import torch

    from dotcache_amd.projection import GroupedWeight, project

    M, K, N, gs = 1100, 320, 1100, 64
    codes, scales, biases, dense = make(N, K, gs, True, 3, "cuda")
    w = GroupedWeight.from_codes(codes, scales, biases, group_size=gs)
    r = np.random.default_rng(3)
    size = 2.0 ** r.integers(-30, 31, size=(M, 1)) if dtype == "bf16" else np.ones((M, 1))
    x = torch.from_numpy((r.normal(size=(M, K)) * size).astype(np.float32)).to(_dt(dtype)).cuda()
    x[5] = 0
    got, xs = project(x, w).double().cpu().numpy(), x.double().cpu().numpy()
    want = xs @ dense.T
    terms = np.abs(xs) @ np.abs(dense).T
    # (below 2^-14 fp16 keeps steps of 2^-24: half of one for a weight near 0)
    bound = (2.0 ** -11 + (K + 8) * 2.0 ** -23) * terms + 2.0 ** -25 * np.abs(xs).sum(1, keepdims=True) + HALF[dtype] * np.abs(want)
    assert np.all(np.abs(got - want) <= bound * (1 + 2.0 ** -20) + 1e-30), float(np.nanmax(np.abs(got - want) / (bound + 1e-30)))
    x[7, 3], x[9, 319] = float("inf"), float("nan")
    bad = project(x, w)
    rows = [i for i in range(M) if i not in (7, 9)]
    assert torch.equal(bad[rows], torch.from_numpy(got).to(bad.dtype).cuda()[rows]) and not torch.isfinite(bad[[7, 9]]).any()


def test_tiles_replay():
    import torch

    from dotcache_amd.projection import project

    x, w, want, dense = exact_case(1030, 256, 1100, 64, True, "bf16", 4)
    held, out = x.clone(), torch.zeros_like(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        project(held, w, out=out)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        project(held, w, out=out)
    for f in (2.0 ** 40, 0.5, 1.0, -(2.0 ** -50)):
        held.copy_(x * f)
        graph.replay()
        assert torch.equal(out, (x.double() * f @ dense.t().contiguous()).to(out.dtype))
        out.zero_()
        torch.cuda.synchronize()
