"""Operators of the cache's write and read path, as cases: what stands between
a layer's projections and its attention over compressed pages.

``rotate``  per-head norms of queries and keys with the position rotation
            (``norm_rotate``)
``append``  the same on the way into the pages: rotated queries out, rotated
            keys and plain values encoded into their pages in one call
            (``append_rotary_with``); the pass reads the pages it wrote back
            as the values they stand for
``read``    tokens of compressed pages as dense rows (``read_tokens_with``)
``attend``  attention of a chunk of new tokens of every sequence over its
            pages, causal among the new ones (``attend_chunk``)

Page formats are written "m3" (fp16 rows) or "<a|s><bits>g<group>" (grouped
affine or symmetric codes), for instance "a4g32".  Inputs are made on the GPU
from the seed alone; where ``own`` is false everything is computed by
elementary torch operations.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_POSITIONS = 40960  # positions that the rotation's table covers
_EPS = 1e-6  # of the norms


def _parse(fmt: str) -> tuple[str, int, int]:
    """(scheme, bits, group): scheme "m3", "a" or "s"."""
    if fmt == "m3":
        return "m3", 0, 32
    bits, group = fmt[1:].split("g")
    return fmt[0], int(bits), int(group)


def _token_bytes(fmt: str, hd: int) -> int:
    scheme, bits, group = _parse(fmt)
    if scheme == "m3":
        return 2 * hd
    return -(-hd // group) * (group * bits // 8 + (4 if scheme == "a" else 2))


# ---- the cases ------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # The new token of each of 16 sequences of a 7B-shaped layer (28 query
        # and 4 KV heads): the smallest call, once per layer and step.
        {"name": "rotate_decode_b16", "kind": "rotate", "tokens": 16, "kv_heads": 4, "q_per_kv": 7, "hd": 128,
         "rotary": 128, "interleaved": False, "norm": True, "dtype": "bf16"},
        # A long prompt of the same layer.
        {"name": "rotate_prompt_16k", "kind": "rotate", "tokens": 16384, "kv_heads": 4, "q_per_kv": 7, "hd": 128,
         "rotary": 128, "interleaved": False, "norm": True, "dtype": "bf16"},
        # One decode step of 64 sequences into 4-bit pages.
        {"name": "append_decode_b64", "kind": "append", "batch": 64, "tokens": 1, "kv_heads": 4, "q_per_kv": 7, "hd": 128,
         "rotary": 128, "interleaved": False, "norm": True, "dtype": "bf16", "page": 64, "key": "a4g32", "value": "s4g32"},
        # A prompt's chunk of four sequences: exact keys, 4-bit values.
        {"name": "append_chunk_b4_4k", "kind": "append", "batch": 4, "tokens": 4096, "kv_heads": 4, "q_per_kv": 7,
         "hd": 128, "rotary": 128, "interleaved": False, "norm": True, "dtype": "bf16", "page": 64, "key": "m3",
         "value": "s4g32"},
        # An odd head_dim with a partial, interleaved rotation and no norms, 8-bit keys.
        {"name": "append_hd96_b3", "kind": "append", "batch": 3, "tokens": 777, "kv_heads": 6, "q_per_kv": 2, "hd": 96,
         "rotary": 48, "interleaved": True, "norm": False, "dtype": "f16", "page": 64, "key": "s8g32", "value": "a4g32"},
        # One block of a prefix, handed on as dense rows.
        {"name": "read_block", "kind": "read", "batch": 1, "tokens": 64, "kv_heads": 4, "hd": 128, "dtype": "bf16",
         "page": 64, "key": "a4g32", "value": "a4g32"},
        # The whole cache of 8 sequences.
        {"name": "read_b8_16k", "kind": "read", "batch": 8, "tokens": 16384, "kv_heads": 4, "hd": 128, "dtype": "bf16",
         "page": 64, "key": "a4g32", "value": "a4g32"},
        # Speculative decoding: five drafted tokens of each of four sequences
        # of very different lengths are verified.
        {"name": "verify_b4_128k", "kind": "attend", "batch": 4, "new": 5, "new_low": 5, "context": 131072,
         "context_low": 1024, "kv_heads": 4, "q_per_kv": 7, "hd": 128, "page": 64, "key": "a4g32", "value": "a4g32",
         "dtype": "bf16"},
        # A prompt's second chunk at a small model's shape.
        {"name": "chunk_512_of_4k", "kind": "attend", "batch": 1, "new": 512, "new_low": 512, "context": 4096,
         "context_low": 4096, "kv_heads": 8, "q_per_kv": 4, "hd": 64, "page": 64, "key": "a4g32", "value": "a4g32",
         "dtype": "f16"},
        # The largest: a long prompt's last chunk, exact keys and 4-bit values.
        {"name": "chunk_2k_of_16k", "kind": "attend", "batch": 2, "new": 2048, "new_low": 2048, "context": 16384,
         "context_low": 16384, "kv_heads": 4, "q_per_kv": 7, "hd": 128, "page": 64, "key": "m3", "value": "s4g32",
         "dtype": "bf16"},
        # A serving engine's mixed batch: decodes and prompt chunks of 1 to 700
        # tokens in one call, head_dim 256, pages of 128 tokens.
        {"name": "mixed_b12_hd256", "kind": "attend", "batch": 12, "new": 700, "new_low": 1, "context": 8192,
         "context_low": 700, "kv_heads": 4, "q_per_kv": 4, "hd": 256, "page": 128, "key": "a4g32", "value": "a4g32",
         "dtype": "bf16"},
        # fp32 throughout, odd sizes, a head_dim that is no power of two.
        {"name": "chunk_f32_hd96", "kind": "attend", "batch": 3, "new": 61, "new_low": 61, "context": 1001,
         "context_low": 1001, "kv_heads": 6, "q_per_kv": 2, "hd": 96, "page": 48, "key": "s8g32", "value": "a4g32",
         "dtype": "f32"},
    ]


def draw(rng: random.Random) -> dict:
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))

    kind = rng.choice(["rotate", "append", "append", "read", "attend", "attend", "attend"])
    hd = rng.choice([64, 96, 128, 128, 256])
    case = {"kind": kind, "hd": hd, "kv_heads": rng.choice([1, 2, 4, 8])}
    formats = ["a4g32", "s4g32", "m3", "a8g32", "s8g64", "a4g64"]
    if kind != "rotate":
        case.update(page=rng.choice([16, 32, 64, 64, 128]), key=rng.choice(formats), value=rng.choice(formats),
                    batch=size(1, 64 if kind != "attend" else 24))
    if kind != "read":
        case["q_per_kv"] = rng.choice([1, 2, 3, 4, 6, 7, 8, 16])
    if kind in ("rotate", "append"):
        case.update(rotary=rng.choice([hd, hd, hd // 2]), interleaved=rng.random() < 0.3, norm=rng.random() < 0.6,
                    dtype=rng.choice(["bf16", "bf16", "f16"] + ["f32"] * (kind == "rotate")))
        row = case["kv_heads"] * (case["q_per_kv"] + 2) * hd * case.get("batch", 1)
        case["tokens"] = size(1, max(1, min(16384, 16384 * 36 * 128 // row)))
    elif kind == "read":
        case["dtype"] = rng.choice(["bf16", "f16"])
        case["tokens"] = size(1, max(1, min(32768, (1 << 26) // (case["batch"] * case["kv_heads"] * hd))))
    else:
        case["dtype"] = rng.choice(["bf16", "bf16", "f16", "f32"])
        if case["dtype"] == "f32":
            case.update(key=rng.choice(formats[:4]), value=rng.choice(formats[:4]))
        streams = case["batch"] * case["kv_heads"]
        case["context"] = size(1, min(131072, (1 << 26) // (streams * hd)))
        case["context_low"] = rng.choice([case["context"], max(1, case["context"] // 8)])
        # an eighth of the largest listed case's products
        rows = (1 << 35) // (streams * case["q_per_kv"] * hd * case["context"])
        case["new"] = size(1, max(1, min(case["context_low"], 2048, rows)))
        case["new_low"] = rng.choice([1, case["new"], case["new"]])
    return case


# ---- seeded inputs ----------------------------------------------------------------
def _gen(seed: int, tag: int):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + tag)
    return g


def _randn(seed: int, tag: int, *shape):
    return torch.randn(shape, generator=_gen(seed, tag), device="cuda")


def _spread(low: int, high: int, count: int, salt: int) -> list[int]:
    """``count`` sizes between low and high, spread over the logarithm and
    fixed by the case: the first is the largest."""
    r = random.Random(low * 31 + high * 7919 + salt)
    lo, hi = math.log(low), math.log(high)
    return [high] + [min(high, max(low, int(math.exp(r.uniform(lo, hi))))) for _ in range(count - 1)]


def _attend_lens(case: dict) -> tuple[list[int], list[int]]:
    """(new tokens, context length with them) of every sequence."""
    ctx = _spread(case["context_low"], case["context"], case["batch"], 1)
    new = _spread(case["new_low"], case["new"], case["batch"], 2)
    return [min(n, c) for n, c in zip(new, ctx)], ctx


def _inv_freq(case: dict):
    rd = case["rotary"]
    return 1.0 / (1000000.0 ** (np.arange(0, rd, 2, dtype=np.float64) / rd))


def _quotient(a, b):
    """The correctly rounded fp32 quotient of two fp32 tensors."""
    return (a.double() / b.double()).float()


def _encode(x, fmt: str):
    """Codes (int32), fp16 scale and fp16 bias of fp32 rows ``x [..., hd]`` in
    groups ``[..., G, group]`` by the page format's definition."""
    scheme, bits, group = _parse(fmt)
    g = torch.nn.functional.pad(x, (0, -x.shape[-1] % group)).unflatten(-1, (-1, group))
    if scheme == "a":
        top = float((1 << bits) - 1)
        lo = g.amin(-1, keepdim=True)
        scale = _quotient(g.amax(-1, keepdim=True) - lo, torch.tensor(top, device=x.device)).clamp_min(1e-8)
        codes = torch.round(_quotient(g - lo, scale)).clamp(0, top)
        return codes.int(), scale.half(), lo.half()
    qmax = float((1 << (bits - 1)) - 1)
    scale = _quotient(g.abs().amax(-1, keepdim=True), torch.tensor(max(qmax, 1.0), device=x.device)).clamp_min(1e-8)
    codes = torch.round(_quotient(g, scale)).clamp(-qmax, qmax) + qmax
    return codes.int(), scale.half(), None


def _values(codes, scale, bias, fmt: str, hd: int):
    """fp32 rows that codes, scales and biases stand for."""
    _, bits, _ = _parse(fmt)
    if bias is None:
        x = (codes - ((1 << (bits - 1)) - 1)).float() * scale.float()
    else:
        x = codes.float() * scale.float() + bias.float()
    return x.flatten(-2)[..., :hd]


def _pages_of(x, fmt: str, page: int, lens):
    """What a cache holds for rows ``x [B, H, T, hd]``: packed words, scales
    and biases (or fp16 rows), and the last page of every sequence exact, as a
    cache keeps a page that still fills."""
    hd = x.shape[-1]
    tail_at = (torch.tensor(lens, device="cuda") - 1) // page * page
    held = {"fmt": fmt, "hd": hd, "tail_at": tail_at, "page": page}
    if fmt == "m3":
        held["rows"] = x.half()
        return held
    _, bits, _ = _parse(fmt)
    codes, scale, bias = _encode(x, fmt)
    per = 32 // bits
    shifts = torch.arange(per, device="cuda", dtype=torch.int64) * bits
    words = (codes.unflatten(-1, (-1, per)).long() << shifts).sum(-1)
    held.update(words=(words - ((words >> 31) << 32)).int(), scale=scale, bias=bias)
    at = (tail_at[:, None] + torch.arange(page, device="cuda"))[:, None, :, None].clamp(max=x.shape[2] - 1)
    held["tail"] = torch.gather(x, 2, at.expand(x.shape[0], x.shape[1], page, hd)).half()
    return held


def _held_rows(held: dict):
    """fp32 rows ``[B, H, T, hd]`` of held pages."""
    if held["fmt"] == "m3":
        return held["rows"].float()
    _, bits, _ = _parse(held["fmt"])
    shifts = torch.arange(32 // bits, device="cuda", dtype=torch.int32) * bits
    codes = ((held["words"][..., None] >> shifts) & ((1 << bits) - 1)).flatten(-2)
    x = _values(codes, held["scale"], held["bias"], held["fmt"], held["hd"])
    T, page = x.shape[2], held["page"]
    x = torch.nn.functional.pad(x, (0, 0, 0, page))
    at = (held["tail_at"][:, None] + torch.arange(page, device="cuda"))[:, None, :, None].expand(held["tail"].shape)
    return x.scatter(2, at, held["tail"].float())[:, :, :T]


def _own_pool(case: dict, fmt: str, pages: int):
    from dotcache_amd.page_pool import DevicePagePool, PoolGeometry, page_format_of

    scheme, bits, group = _parse(fmt)
    form = page_format_of("M3" if scheme == "m3" else "M0", "symmetric" if scheme == "s" else "affine", bits or 4)
    geo = PoolGeometry(case["hd"], group, case["page"])
    return DevicePagePool(geo, reserve_bytes=pages * case["page"] * 2 * case["hd"] + (1 << 20), reserve_pages=pages + 16), form


def _own_filled(case: dict, fmt: str, x, lens, seed: int, tail: bool):
    """A pool that holds rows ``x [B, H, T, hd]``, its pages in any order, and
    the page table ``[B, H, pages]``; the last page of a sequence exact."""
    B, H, T, hd = x.shape
    P = case["page"]
    W = -(-T // P)
    pool, form = _own_pool(case, fmt, B * H * W + B * H)
    body = pool.allocate(*form, B * H * W, tokens=P)
    r = np.random.default_rng(seed)
    table = r.permutation(body).reshape(B, H, W).astype(np.int32)
    last = (np.asarray(lens) - 1) // P
    if tail and fmt != "m3":
        table[np.arange(B), :, last] = pool.allocate(0, 0, B * H, tokens=P).reshape(B, H)
    pool.set_tokens(table[np.arange(B), :, last].ravel(), np.repeat(np.asarray(lens) - last * P, H))
    ids = torch.from_numpy(table).cuda()
    token = torch.arange(T, device="cuda")
    pool.encode_rows(x.reshape(B * H * T, hd), ids[:, :, token // P].reshape(-1).int(),
                     (token % P).int().expand(B, H, T).reshape(-1))
    return pool, ids, table


# ---- rotate -------------------------------------------------------------------------
def _rotated(x, weight, positions, table, case: dict, dtype):
    """Normed and rotated rows of ``x [T, heads, hd]`` in ``dtype``."""
    y = x.to(dtype)
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + _EPS) * weight.to(dtype)
    rd = case["rotary"]
    cos, sin = (t[:, None, :].to(dtype) for t in table[positions.long()].split(rd // 2, dim=-1))
    if case["interleaved"]:
        a, b = y[..., 0:rd:2], y[..., 1:rd:2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = y[..., : rd // 2], y[..., rd // 2: rd]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([r, y[..., rd:]], dim=-1)


def _rotate_inputs(case: dict, seed: int, tokens: int) -> dict:
    """One projection's output, [tokens, (Hq + 2 Hkv) hd], of which queries,
    keys and values are views; positions, norm weights and the table."""
    H, hd, dtype = case["kv_heads"], case["hd"], _DTYPES[case["dtype"]]
    heads = H * case["q_per_kv"]
    fused = _randn(seed, 1, tokens, heads + 2 * H, hd)
    fused = (fused * torch.exp(0.5 * _randn(seed, 2, 1, heads + 2 * H, hd))).to(dtype)  # channels differ in size
    angles = torch.arange(_POSITIONS, dtype=torch.float64, device="cuda")[:, None] * torch.from_numpy(_inv_freq(case)).cuda()
    state = {"case": case, "q": fused[:, :heads], "k": fused[:, heads: heads + H], "v": fused[:, heads + H:],
             "table": torch.cat([angles.cos(), angles.sin()], dim=-1).float(), "qw": None, "kw": None}
    if case["norm"]:
        state["qw"], state["kw"] = (1.0 + 0.2 * _randn(seed, 3 + i, hd) for i in range(2))
    return state


def _own_rotary(case: dict):
    from dotcache_amd.rotary import RotaryTable

    return RotaryTable(case["hd"], _POSITIONS, rotary_dim=case["rotary"], inv_freq=_inv_freq(case),
                       interleaved=case["interleaved"])


def _prepare_rotate(case: dict, seed: int) -> dict:
    T = case["tokens"]
    state = _rotate_inputs(case, seed, T)
    if T > 64:  # a prompt's positions in order, or one position of each sequence
        state["positions"] = torch.arange(T, device="cuda", dtype=torch.int32) + seed % 1000
    else:
        state["positions"] = torch.randint(0, _POSITIONS, (T,), generator=_gen(seed, 9), device="cuda", dtype=torch.int32)
    if own:
        state["rotary"] = _own_rotary(case)
    return state


def _run_rotate(state: dict):
    if own:
        from dotcache_amd.rotary import norm_rotate

        return norm_rotate(state["q"], state["k"], state["positions"], state["rotary"], q_weight=state["qw"],
                           k_weight=state["kw"], eps=_EPS)
    case = state["case"]
    return tuple(_rotated(state[x], state[x + "w"], state["positions"], state["table"], case, torch.float32)
                 .to(state[x].dtype) for x in ("q", "k"))


def _exact_rotation(x, weight, positions, case: dict):
    """The same in 64 bits: pairs as complex numbers, turned by their angle."""
    y = x.double()
    if weight is not None:
        y = y / torch.linalg.vector_norm(torch.cat([y, torch.full_like(y[..., :1], math.sqrt(_EPS * y.shape[-1]))], -1),
                                         dim=-1, keepdim=True) * math.sqrt(y.shape[-1]) * weight.double()
    rd = case["rotary"]
    head, rest = y[..., :rd], y[..., rd:]
    pairs = head.unflatten(-1, (-1, 2)) if case["interleaved"] else head.unflatten(-1, (2, -1)).transpose(-1, -2)
    angle = positions.double()[:, None, None] * torch.from_numpy(_inv_freq(case)).cuda()
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.ones_like(angle), angle))
    turned = turned if case["interleaved"] else turned.transpose(-1, -2)
    return torch.cat([turned.flatten(-2), rest], dim=-1)


def _exact_rotate(case: dict, seed: int):
    s = _prepare_rotate(case, seed)
    return tuple(_exact_rotation(s[x], s[x + "w"], s["positions"], case) for x in ("q", "k"))


# ---- append -------------------------------------------------------------------------
def _prepare_append(case: dict, seed: int) -> dict:
    """``tokens`` new tokens of each sequence, token-major; every sequence
    starts at its own place in its pages and at its own position."""
    B, n, H, P = case["batch"], case["tokens"], case["kv_heads"], case["page"]
    state = _rotate_inputs(case, seed, B * n)
    r = np.random.default_rng(seed)
    first = r.integers(0, P, B) if n > 1 else r.integers(0, 8 * P, B)
    token = (first[:, None] + np.arange(n)).astype(np.int32)
    start = r.integers(0, _POSITIONS - n, B)
    state["positions"] = torch.from_numpy((start[:, None] + np.arange(n)).astype(np.int32).ravel()).cuda()
    if own:
        W = int(token.max()) // P + 1
        state["pools"], ids = [], []
        for fmt in (case["key"], case["value"]):
            pool, form = _own_pool(case, fmt, B * H * W)
            ids.append(r.permutation(pool.allocate(*form, B * H * W, tokens=P)).reshape(B, H, W))
            state["pools"].append(pool)
        state["tables"] = torch.from_numpy(np.stack(ids).astype(np.int32)).cuda()
        state["row"] = torch.from_numpy(np.repeat(np.arange(B, dtype=np.int32), n)).cuda()
        state["token"] = torch.from_numpy(token.ravel()).cuda()
        state["rotary"] = _own_rotary(case)
    return state


def _stored(x, fmt: str):
    return x.half().float() if fmt == "m3" else _values(*_encode(x, fmt), fmt, x.shape[-1])


def _run_append(state: dict):
    case = state["case"]
    dtype = state["q"].dtype
    if own:
        k_pool, v_pool = state["pools"]
        q = k_pool.append_rotary_with(v_pool, state["q"], state["k"], state["v"], state["positions"], state["rotary"],
                                      state["tables"], state["row"], state["token"], q_weight=state["qw"],
                                      k_weight=state["kw"], eps=_EPS)
        k, v = k_pool.read_tokens_with(v_pool, state["tables"], state["row"], state["token"], dtype=dtype)
        return q, k, v
    q = _rotated(state["q"], state["qw"], state["positions"], state["table"], case, torch.float32).to(dtype)
    # (codes are values next to a border: the keys in 64 bits, rounded to fp32 once)
    k = _rotated(state["k"], state["kw"], state["positions"], state["table"], case, torch.float64).float()
    return q, _stored(k, case["key"]).to(dtype), _stored(state["v"].float(), case["value"]).to(dtype)


def _exact_stored(x, fmt: str):
    """Values of 64-bit rows in a page: the nearest of the group's levels, with
    the fp16 scale and offset that the page keeps."""
    scheme, bits, group = _parse(fmt)
    if scheme == "m3":
        return x.half().double()
    hd = x.shape[-1]
    g = torch.nn.functional.pad(x, (0, -hd % group)).unflatten(-1, (-1, group))
    low = g.min(-1, keepdim=True).values if scheme == "a" else torch.zeros_like(g[..., :1])
    span = (g.max(-1, keepdim=True).values - low) / (2 ** bits - 1) if scheme == "a" \
        else g.abs().max(-1, keepdim=True).values / (2 ** (bits - 1) - 1)
    span = torch.maximum(span, torch.full_like(span, 1e-8)).float().double()  # (the format's scales are fp32 numbers)
    return (torch.round(((g - low) / span).float()).double() * span.half().double() + low.half().double()).flatten(-2)[..., :hd]


def _exact_append(case: dict, seed: int):
    s = _prepare_append(case, seed)
    q, k = (_exact_rotation(s[x], s[x + "w"], s["positions"], case) for x in ("q", "k"))
    return q, _exact_stored(k, case["key"]), _exact_stored(s["v"].double(), case["value"])


# ---- read ---------------------------------------------------------------------------
def _cache_rows(case: dict, seed: int, tokens: int):
    """Keys and values [B, H, T, hd] that went into the cache: a few channels
    of each head are much larger than the others."""
    out = []
    for tag in (11, 13):
        x = _randn(seed, tag, case["batch"], case["kv_heads"], tokens, case["hd"])
        x = x * torch.exp(0.6 * _randn(seed, tag + 1, 1, case["kv_heads"], 1, case["hd"]))
        out.append(x.to(torch.bfloat16).float())
    return out


def _prepare_read(case: dict, seed: int) -> dict:
    B, T = case["batch"], case["tokens"]
    rows = _cache_rows(case, seed, T)
    state = {"case": case, "held": [_pages_of(x, f, case["page"], [T] * B) for x, f in zip(rows, (case["key"], case["value"]))]}
    if own:
        filled = [_own_filled(case, f, x, [T] * B, seed + i, True)
                  for i, (x, f) in enumerate(zip(rows, (case["key"], case["value"])))]
        state["pools"] = [f[0] for f in filled]
        state["tables"] = torch.stack([f[1] for f in filled])
        state["row"] = torch.arange(B, device="cuda", dtype=torch.int32).repeat_interleave(T)
        state["token"] = torch.arange(T, device="cuda", dtype=torch.int32).repeat(B)
    return state


def _run_read(state: dict):
    dtype = _DTYPES[state["case"]["dtype"]]
    if own:
        k_pool, v_pool = state["pools"]
        return k_pool.read_tokens_with(v_pool, state["tables"], state["row"], state["token"], dtype=dtype)
    return tuple(_held_rows(h).to(dtype).transpose(1, 2).flatten(0, 1).contiguous() for h in state["held"])


def _exact_held(held: dict, b: int, h: int):
    """One stream's rows in 64 bits, each code cut out of its word."""
    if held["fmt"] == "m3":
        return held["rows"][b, h].double()
    scheme, bits, group = _parse(held["fmt"])
    words = held["words"][b, h].long() & 0xFFFFFFFF
    i = torch.arange(group, device="cuda")
    codes = torch.div(words[..., i * bits // 32], 2 ** (i * bits % 32), rounding_mode="floor") % 2 ** bits
    zero = 0 if scheme == "a" else 2 ** (bits - 1) - 1
    x = (codes - zero).double() * held["scale"][b, h].double()
    if scheme == "a":
        x = x + held["bias"][b, h].double()
    x = x.reshape(x.shape[0], -1)[:, : held["hd"]]
    at = int(held["tail_at"][b])
    n = min(held["page"], x.shape[0] - at)
    x[at: at + n] = held["tail"][b, h, :n].double()
    return x


def _exact_read(case: dict, seed: int):
    s = _prepare_read(case, seed)
    return tuple(torch.stack([torch.stack([_exact_held(h, b, j) for j in range(case["kv_heads"])], 1)
                              for b in range(case["batch"])]).flatten(0, 1) for h in s["held"])


# ---- attend -------------------------------------------------------------------------
def _prepare_attend(case: dict, seed: int) -> dict:
    new, ctx = _attend_lens(case)
    B, Hq, hd = case["batch"], case["kv_heads"] * case["q_per_kv"], case["hd"]
    rows = _cache_rows(case, seed, max(ctx))
    state = {"case": case, "held": [_pages_of(x, f, case["page"], ctx) for x, f in zip(rows, (case["key"], case["value"]))]}
    state["q"] = _randn(seed, 21, sum(new), Hq, hd).to(_DTYPES[case["dtype"]])
    state["scale"] = 1.0 / math.sqrt(hd)
    state["new"], state["ctx"] = (torch.tensor(x, device="cuda") for x in (new, ctx))
    start = np.concatenate([[0], np.cumsum(new)])[:-1]
    state["from"] = torch.from_numpy(start[:, None] + np.minimum(np.arange(max(new)), np.asarray(new)[:, None] - 1)).cuda()
    state["to"] = torch.from_numpy(np.concatenate([b * max(new) + np.arange(n) for b, n in enumerate(new)])).cuda()
    if own:
        from dotcache_amd.chunk import plan_chunk

        filled = [_own_filled(case, f, x, ctx, seed + i, True)
                  for i, (x, f) in enumerate(zip(rows, (case["key"], case["value"])))]
        state["pools"] = [f[0] for f in filled]
        state["tables"] = [f[1] for f in filled]
        state["plan"] = plan_chunk(filled[0][0], filled[1][0], new, ctx, kv_heads=case["kv_heads"],
                                   q_per_kv=case["q_per_kv"], dtype=state["q"].dtype)
    return state


def _run_attend(state: dict):
    case = state["case"]
    if own:
        from dotcache_amd.chunk import attend_chunk

        (k_pool, v_pool), (kt, vt) = state["pools"], state["tables"]
        return attend_chunk(k_pool, kt, v_pool, vt, state["q"], state["plan"], query_scale=state["scale"])
    H, n_q, hd = case["kv_heads"], case["q_per_kv"], case["hd"]
    k, v = (_held_rows(h) for h in state["held"])
    B, N = state["from"].shape
    # [B, H, new * n_q, hd]: every sequence padded to the longest
    q = state["q"][state["from"]].float().reshape(B, N, H, n_q, hd).transpose(1, 2).reshape(B, H, N * n_q, hd)
    s = torch.matmul(q * state["scale"], k.transpose(-1, -2).contiguous())
    last = (state["ctx"] - state["new"])[:, None] + torch.arange(N, device="cuda")  # the last token a row sees
    last = torch.minimum(last, state["ctx"][:, None] - 1)[:, None, :, None].expand(B, 1, N, n_q).reshape(B, 1, N * n_q, 1)
    s = s.masked_fill_(torch.arange(k.shape[2], device="cuda") > last, -math.inf)
    p = s.sub_(s.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    o = o.reshape(B, H, N, n_q, hd).transpose(1, 2).reshape(B * N, H * n_q, hd)
    return o[state["to"]].to(state["q"].dtype)


def _exact_attend(case: dict, seed: int):
    s = _prepare_attend(case, seed)
    new, ctx = _attend_lens(case)
    n_q, out, t0 = case["q_per_kv"], torch.empty_like(s["q"], dtype=torch.float64), 0
    for b in range(case["batch"]):
        n, c = new[b], ctx[b]
        sees = torch.arange(c, device="cuda")[None, :] <= torch.arange(c - n, c, device="cuda")[:, None]
        for h in range(case["kv_heads"]):
            k, v = (_exact_held(x, b, h)[:c] for x in s["held"])
            kt = k.t().contiguous()
            for j in range(h * n_q, (h + 1) * n_q):
                logits = (s["q"][t0: t0 + n, j].double() @ kt) * s["scale"]
                w = torch.softmax(torch.where(sees, logits, torch.full_like(logits, -math.inf)), dim=-1)
                out[t0: t0 + n, j] = w @ v
        t0 += n
    return out


# ---- the interface ------------------------------------------------------------------
def prepare(case: dict, seed: int) -> dict:
    return {"rotate": _prepare_rotate, "append": _prepare_append, "read": _prepare_read,
            "attend": _prepare_attend}[case["kind"]](case, seed)


def run(state: dict):
    return {"rotate": _run_rotate, "append": _run_append, "read": _run_read, "attend": _run_attend}[state["case"]["kind"]](state)


def exact(case: dict, seed: int):
    return {"rotate": _exact_rotate, "append": _exact_append, "read": _exact_read,
            "attend": _exact_attend}[case["kind"]](case, seed)


def work(case: dict) -> dict:
    kind, H, hd = case["kind"], case["kv_heads"], case["hd"]
    e = 4 if case["dtype"] == "f32" else 2
    stored = sum(_token_bytes(case[x], hd) for x in ("key", "value")) if kind != "rotate" else 0
    if kind == "attend":
        new, ctx = _attend_lens(case)
        pairs = sum(n * (c - n) + n * (n + 1) // 2 for n, c in zip(new, ctx))
        return {"bytes": H * (sum(ctx) * stored + 2 * sum(new) * case["q_per_kv"] * hd * e),
                "flops": 4 * pairs * H * case["q_per_kv"] * hd}
    T = case["tokens"] * case.get("batch", 1)
    if kind == "read":
        return {"bytes": T * H * (stored + 2 * hd * e), "flops": 4 * T * H * hd}
    heads = H * (case["q_per_kv"] + 1)  # queries and keys
    table = 4 * T * case["rotary"]
    if kind == "rotate":
        return {"bytes": 2 * T * heads * hd * e + table, "flops": 8 * T * heads * hd}
    # queries and keys in, queries out, values in; the pages written, read again, and their values out
    moved = (H * (2 * case["q_per_kv"] + 2) * hd * e) + 2 * H * stored + 2 * H * hd * e
    return {"bytes": T * moved + table, "flops": T * (8 * heads + 12 * H) * hd}
