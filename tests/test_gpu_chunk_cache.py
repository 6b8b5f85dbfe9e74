"""The caches' chunk calls together, as a model's layer makes them: norm, rotate
and append a prompt's chunks, attend them, verify drafted tokens, decode, read
the tokens back -- against the fp64 formulas on the pages' own values."""
import numpy as np
import pytest

from dotcache_amd.config import DotCacheConfig
from tests.test_gpu_chunk import _bound
from tests.test_gpu_kv_cache import KERNEL_TOL

pytestmark = pytest.mark.gpu


def _formula(x, w, eps, rotary, positions):
    """Norm and half-split rotation of x [tokens, heads, hd] in fp64, and the
    largest |channel| of each result before its own sums (for tolerances)."""
    y = x.astype(np.float64)
    if w is not None:
        y = y / np.sqrt(np.mean(y * y, axis=-1, keepdims=True) + eps) * w.astype(np.float64)
    rd = rotary.rotary_dim
    row = rotary.table.double().cpu().numpy()[positions]
    c, s = row[:, None, : rd // 2], row[:, None, rd // 2:]
    a, b = y[..., : rd // 2].copy(), y[..., rd // 2: rd].copy()
    y[..., : rd // 2], y[..., rd // 2: rd] = a * c - b * s, b * c + a * s
    return y, np.max(np.abs(np.concatenate([a, b, y], -1)), axis=-1, keepdims=True)


def _attended(q, k, v, n, scale, dtype):
    """fp64 attention of q [n, Hq, hd] over k, v [H, T, hd], the bound beside it."""
    H, T, hd = k.shape
    Hq = q.shape[1]
    out, size, logit = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:2])
    for i in range(n):
        m = T - n + i + 1
        for j in range(Hq):
            h = j // (Hq // H)
            s = scale * (k[h, :m] @ q[i, j])
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, j], size[i, j] = p @ v[h, :m], p @ np.abs(v[h, :m])
            logit[i, j] = scale * np.max(np.abs(k[h, :m]) @ np.abs(q[i, j]))
    return out, _bound(dtype, out, size, logit, T, hd, np.max(np.abs(v)))


def _check_attend(got, q, k, v, scale, dtype):
    want, bound = _attended(q, k, v, q.shape[0], scale, dtype)
    err = np.abs(got.double().cpu().numpy() - want)
    assert np.all(err <= bound), float(np.max(err / bound))


def _check_queries(out, x, w, eps, rotary, positions, dtype):
    """fp32 arithmetic (a norm's sum of hd squares, a handful of roundings
    after it) and the output's own rounding."""
    want, size = _formula(x, w, eps, rotary, positions)
    half = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
    bound = half * np.abs(want) * 1.01 + (x.shape[-1] + 16) * 2.0 ** -24 * size + (2.0 ** -25 if dtype == "f16" else 0)
    err = np.abs(out.double().cpu().numpy() - want)
    assert np.all(err <= bound), float(np.max(err / bound))


def _dt(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


@pytest.mark.parametrize("batch,hd,P,dtype,mode,gain", [
    (1, 64, 16, "bf16", "M0", True), (2, 128, 32, "f16", "M0", True), (3, 96, 16, "f32", "M0", False),
    (2, 64, 16, "bf16", "M3", True), (1, 64, 16, "f32", "strict", True)])
def test_a_layer_of_the_paged_cache(batch, hd, P, dtype, mode, gain):
    import torch

    from dotcache_amd.kv_cache import DevicePagedKVCache
    from dotcache_amd.rotary import RotaryTable

    H, Hq, eps, scale = 2, 6, 1e-6, 1.0 / np.sqrt(hd)
    print(f"paged layer batch {batch} hd {hd} {dtype} {mode}", flush=True)
    rng = np.random.default_rng(hd + batch)
    how = dict(key_policy_tier="strict") if mode == "strict" else dict(default_mode_k=mode)  # (strict: by the page's age and rows)
    cfg = DotCacheConfig(head_dim=hd, group_size=32, tokens_per_page=P, bits_k=4, bits_v=4, default_mode_v="M0", **how)
    cache = DevicePagedKVCache(cfg, num_hidden_layers=2, num_attention_heads=Hq, num_key_value_heads=H, batch_size=batch)
    plain = DevicePagedKVCache(cfg, num_hidden_layers=2, num_attention_heads=Hq, num_key_value_heads=H, batch_size=batch)
    rotary = RotaryTable(hd, 256)
    w = [torch.from_numpy((1 + 0.2 * rng.normal(size=hd)).astype(np.float32)).cuda() if gain else None for _ in range(2)]
    wn = [None if x is None else x.cpu().numpy() for x in w]
    at = 0
    # within the first page; past it and over whole pages; one token; to a page's end; drafted tokens
    for n in (P - 3, 2 * P + 7, 1, P - 5, 5):
        q, k, v = (torch.from_numpy(rng.normal(size=(batch, n, h, hd)).astype(np.float32)).to(_dt(dtype)).cuda().transpose(1, 2)
                   for h in (Hq, H, H))
        out = cache.append_rotated(1, q, k, v, at, rotary, q_weight=w[0], k_weight=w[1], eps=eps)
        assert out.shape == q.shape and out.dtype == q.dtype
        pos = np.arange(at, at + n)
        rows = []
        for b in range(batch):
            _check_queries(out[b].transpose(0, 1), q[b].transpose(0, 1).float().cpu().numpy(), wn[0], eps, rotary, pos, dtype)
            rows.append(_formula(k[b].transpose(0, 1).float().cpu().numpy(), wn[1], eps, rotary, pos)[0].astype(np.float32))
        # the fp64 formula's rows through append_step: the same cache, byte for byte
        plain.append_step(1, np.stack(rows).transpose(0, 2, 1, 3), v.float(), at)
        at += n
        assert cache.sequence_length(1) == at
        kd, vd = cache.read_layer(1)
        assert kd.shape == (batch, H, at, hd)
        for x, y in zip((kd, vd), plain.read_layer(1)):
            assert torch.equal(x, y)
        for kind in ("K", "V"):
            pages = cache.page_ids(1, batch - 1, 1, kind)
            assert len(pages) == at // P
            if pages:
                a, b = (c.page(1, batch - 1, 1, len(pages) - 1, kind) for c in (cache, plain))
                assert a.header == b.header
        got = cache.attend_chunk(1, out, query_scale=scale)
        assert got.shape == q.shape and got.dtype == q.dtype
        for b in range(batch):
            _check_attend(got[b].transpose(0, 1), out[b].transpose(0, 1).double().cpu().numpy(), kd[b].double().cpu().numpy(),
                          vd[b].double().cpu().numpy(), scale, dtype)
    # one token at a time: the decode of the same queries
    q = out[:, :, -1].contiguous()
    one = cache.attend_chunk(1, q.unsqueeze(2), query_scale=scale)[:, :, 0].float().cpu().numpy()
    dec = cache.decode_layer(1, q, query_scale=scale).cpu().numpy()
    for b in range(batch):
        _, bound = _attended(q[b:b + 1].double().cpu().numpy(), kd[b].double().cpu().numpy(), vd[b].double().cpu().numpy(), 1, scale, dtype)
        assert np.all(np.abs(one[b] - dec[b]) <= bound[0] + KERNEL_TOL * np.max(np.abs(vd[b].double().cpu().numpy())))
    # query heads in another order
    order = np.array([1, 0, 1, 0, 0, 1])
    perm = np.argsort(order, kind="stable")
    got = cache.attend_chunk(1, out, order, query_scale=scale)
    same = cache.attend_chunk(1, out[:, perm.tolist()].contiguous(), query_scale=scale)
    assert torch.equal(got[:, perm.tolist()], same)
    assert cache.sequence_length(0) == 0


@pytest.mark.parametrize("hd,dtype", [(64, "bf16"), (128, "f32")])
def test_a_serving_step_over_blocks(hd, dtype):
    """Prompts of two sequences in chunks with a third decoding, blocks that
    fill and one that is reused, against a cache written by write_slots."""
    import torch

    from dotcache_amd.block_cache import DeviceVllmPagedKVCache
    from dotcache_amd.rotary import RotaryTable

    H, Hq, P, eps, scale = 2, 4, 16, 1e-6, 1.0 / np.sqrt(hd)
    print(f"blocks hd {hd} {dtype}", flush=True)
    rng = np.random.default_rng(hd)
    cfg = DotCacheConfig(head_dim=hd, group_size=32, tokens_per_page=P, bits_k=4, bits_v=4)
    make = lambda: DeviceVllmPagedKVCache(config=cfg, num_hidden_layers=1, num_attention_heads=Hq,  # noqa: E731
                                          num_key_value_heads=H, block_size=P)
    cache, plain = make(), make()
    rotary = RotaryTable(hd, 128)
    w = torch.from_numpy((1 + 0.2 * rng.normal(size=(H, hd))).astype(np.float32)).cuda()
    tables = np.array([[5, 1, 9, 2], [7, 3, 11, 0], [4, 6, 8, 10]])
    lens = np.zeros(3, dtype=np.int64)
    for new in ([10, 20, 1], [6, 17, 1], [20, 1, 1], [1, 5, 14]):
        new = np.array(new)
        seq = np.repeat(np.arange(3), new)
        pos = np.concatenate([np.arange(a, a + n) for a, n in zip(lens, new)])
        slots = tables[seq, pos // P] * P + pos % P
        T = int(new.sum())
        q, k, v = (torch.from_numpy(rng.normal(size=(T, h, hd)).astype(np.float32)).to(_dt(dtype)).cuda() for h in (Hq, H, H))
        out = cache.write_slots_rotated(0, q, k, v, slots, pos, rotary, k_weight=w, eps=eps)
        _check_queries(out, q.float().cpu().numpy(), None, eps, rotary, pos, dtype)
        rows = _formula(k.float().cpu().numpy(), w.cpu().numpy(), eps, rotary, pos)[0].astype(np.float32)
        plain.write_slots(0, rows, v.float(), slots)
        lens += new
        got = cache.read_block_tables(0, tables, lens)
        for x, y in zip(got, plain.read_block_tables(0, tables, lens)):
            assert x.shape == (lens.sum(), H, hd) and torch.equal(x, y)
        att = cache.attend_block_tables(0, out, new, tables, lens, query_scale=scale)
        assert att.shape == out.shape and att.dtype == out.dtype
        kd, vd = (x.double().cpu().numpy() for x in got)
        t, r = 0, 0
        for b in range(3):
            _check_attend(att[t: t + new[b]], out[t: t + new[b]].double().cpu().numpy(), kd[r: r + lens[b]].transpose(1, 0, 2),
                          vd[r: r + lens[b]].transpose(1, 0, 2), scale, dtype)
            t, r = t + new[b], r + lens[b]
    # waiting sequences, and a sequence that starts over in a block it had
    q = torch.randn(2, Hq, hd, device="cuda").to(_dt(dtype))
    att = cache.attend_block_tables(0, q, [0, 2, 0], tables, lens, query_scale=scale)
    r = int(lens[0])
    _check_attend(att, q.double().cpu().numpy(), kd[r: r + lens[1]].transpose(1, 0, 2), vd[r: r + lens[1]].transpose(1, 0, 2), scale, dtype)
    k = torch.randn(3, H, hd, device="cuda").to(_dt(dtype))
    cache.write_slots_rotated(0, None, k, k, 5 * P + np.arange(3), np.arange(3), None)
    kd, vd = cache.read_block_tables(0, [[5]], [3], dtype=torch.float32)
    half = k.float().half().float()  # (a live block is an fp16 page)
    assert torch.equal(kd, half) and torch.equal(vd, half)
