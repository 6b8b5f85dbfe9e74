"""Operators of an attention layer whose weights and cache are held in 4 bits,
as cases: the products around the cache, and attention whose scores are not
plain causal ones.

``attend``   attention of new tokens over compressed pages (one token of every
             sequence, drafted tokens, prompt chunks) with scores capped by a
             tanh, lowered by the distance, and with a sliding window (and the
             tokens at a document's start that stay in sight), a prefix that
             sees itself both ways, or several documents in one sequence
             (``plan_chunk`` with a ``ChunkMask``, ``attend_chunk`` with
             ``cap`` and ``slopes``)
``project``  rows times a weight matrix of grouped 4-bit codes
             (``GroupedWeight``, ``project``)

Formats are written "m3" (fp16 rows) or "<a|s><bits>g<group>" (grouped affine or
symmetric codes), for instance "a4g32".  Inputs are made on the GPU from the seed
alone; where ``own`` is false everything is computed by elementary torch
operations.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _parse(fmt: str) -> tuple[str, int, int]:
    """(scheme, bits, group): scheme "m3", "a" or "s"."""
    if fmt == "m3":
        return "m3", 0, 32
    bits, group = fmt[1:].split("g")
    return fmt[0], int(bits), int(group)


def _row_bytes(fmt: str, width: int) -> int:
    scheme, bits, group = _parse(fmt)
    if scheme == "m3":
        return 2 * width
    return -(-width // group) * (group * bits // 8 + (4 if scheme == "a" else 2))


# ---- the cases ------------------------------------------------------------------
# window 0: none; sinks: tokens at a document's start that a window leaves in
# sight; prefix: tokens at a sequence's start that see each other both ways;
# documents: how many a sequence holds; cap 0: none.
_PLAIN = {"window": 0, "sinks": 0, "prefix": 0, "documents": 1, "cap": 0.0, "slopes": False}


def listed() -> list[dict]:
    def attend(name, **k):
        return {"name": name, "kind": "attend", **_PLAIN, **k}

    def project(name, **k):
        return {"name": name, "kind": "project", **k}

    return [
        # The new token of each of 32 sequences in a layer with a sliding window
        # that keeps the first tokens: the smallest attention, where latency counts.
        attend("window_decode_b32", batch=32, new=1, new_low=1, context=32768, context_low=512, kv_heads=4, q_per_kv=7,
               hd=128, page=64, key="a4g32", value="s4g32", dtype="bf16", window=1024, sinks=4),
        # One decode step over whole contexts with capped scores, head_dim 256.
        attend("cap_decode_b8_32k", batch=8, new=1, new_low=1, context=32768, context_low=32768, kv_heads=4, q_per_kv=4,
               hd=256, page=128, key="a4g32", value="a4g32", dtype="bf16", cap=50.0),
        # A prompt's chunk at a small model's shape, scores lowered by distance.
        attend("distance_chunk_1k_of_4k", batch=1, new=1024, new_low=1024, context=4096, context_low=4096, kv_heads=8,
               q_per_kv=4, hd=64, page=64, key="a4g32", value="a4g32", dtype="f16", slopes=True),
        # A prompt packed of 40 documents: exact keys, 4-bit values.
        attend("documents_8k", batch=1, new=8192, new_low=8192, context=8192, context_low=8192, kv_heads=4, q_per_kv=7,
               hd=128, page=64, key="m3", value="s4g32", dtype="bf16", documents=40),
        # Four prompts whose first part (a picture, an encoded text) sees itself
        # both ways; a head_dim that is no power of two, 8-bit keys.
        attend("prefix_b4_hd96", batch=4, new=900, new_low=900, context=900, context_low=900, kv_heads=4, q_per_kv=2,
               hd=96, page=64, key="s8g32", value="a4g32", dtype="f16", prefix=640),
        # The largest: a long prompt's last chunk in a layer with a window and
        # capped scores, head_dim 256.
        attend("window_cap_chunk_2k_of_16k", batch=2, new=2048, new_low=2048, context=16384, context_low=16384,
               kv_heads=4, q_per_kv=4, hd=256, page=128, key="a4g32", value="a4g32", dtype="bf16", window=4096, cap=50.0),
        # Drafted tokens in fp32 with every rule at once and odd sizes.
        attend("verify_f32_hd96", batch=3, new=7, new_low=7, context=1001, context_low=333, kv_heads=6, q_per_kv=2,
               hd=96, page=48, key="s8g32", value="a4g32", dtype="f32", window=301, sinks=5, cap=30.0, slopes=True),
        # The product that makes queries, keys and values of one new token
        # (28 query and 4 KV heads of 128): the smallest call.
        project("project_b1", rows=1, inputs=3584, outputs=4608, weight="a4g64", dtype="bf16"),
        # The product behind the attention for a batch of 16.
        project("project_b16", rows=16, inputs=3584, outputs=3584, weight="s4g32", dtype="f16"),
        # A wide layer for a serving batch.
        project("project_b48_wide", rows=48, inputs=4096, outputs=16384, weight="a4g128", dtype="bf16"),
        # Queries, keys and values of a prompt's chunk.
        project("project_prompt_2k", rows=2048, inputs=3584, outputs=4608, weight="a4g64", dtype="bf16"),
        # fp32 throughout, sizes that fill neither a group nor a tile.
        project("project_f32_odd", rows=5, inputs=1000, outputs=777, weight="a4g32", dtype="f32"),
    ]


def draw(rng: random.Random) -> dict:
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))

    if rng.random() < 0.4:
        rows, inputs = size(1, 4096), size(64, 8192)
        case = {"kind": "project", "rows": rows, "inputs": inputs,
                "weight": rng.choice("as") + "4g" + rng.choice(["32", "64", "128"]),
                "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
        most = (1 << (35 if case["dtype"] != "f32" else 31)) // (rows * inputs)
        case["outputs"] = size(16, max(16, min(32768, most)))
        if rng.random() < 0.5:  # as models have them
            case["inputs"], case["outputs"] = (max(128, x // 128 * 128) for x in (case["inputs"], case["outputs"]))
        return case
    formats = ["a4g32", "s4g32", "m3", "a8g32", "s8g64", "a4g64"]
    case = {"kind": "attend", **_PLAIN, "hd": rng.choice([64, 96, 128, 128, 256]), "kv_heads": rng.choice([1, 2, 4, 8]),
            "q_per_kv": rng.choice([1, 2, 3, 4, 6, 7, 8, 16]), "page": rng.choice([16, 32, 64, 64, 128]),
            "key": rng.choice(formats), "value": rng.choice(formats), "batch": size(1, 32),
            "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    if case["dtype"] == "f32":
        case.update(key=rng.choice(formats[:4]), value=rng.choice(formats[:4]))
    streams = case["batch"] * case["kv_heads"]
    case["context"] = size(1, min(65536, (1 << 26) // (streams * case["hd"])))
    case["context_low"] = rng.choice([case["context"], max(1, case["context"] // 8)])
    rows = (1 << 34) // (streams * case["q_per_kv"] * case["hd"] * case["context"])
    case["new"] = size(1, max(1, min(case["context_low"], 4096, rows)))
    case["new_low"] = rng.choice([1, case["new"], case["new"]])
    if rng.random() < 0.5:
        case.update(window=size(1, case["context"]), sinks=rng.choice([0, 0, 1, 4, 64]))
    if rng.random() < 0.25:
        case["prefix"] = size(1, case["context"])
    if rng.random() < 0.3:
        case["documents"] = size(2, max(2, case["context"] // 4))
    if rng.random() < 0.45:
        case["cap"] = rng.choice([5.0, 30.0, 50.0])
    case["slopes"] = rng.random() < 0.35
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


def _lens(case: dict) -> tuple[list[int], list[int]]:
    """(new tokens, context length with them) of every sequence."""
    ctx = _spread(case["context_low"], case["context"], case["batch"], 1)
    new = _spread(case["new_low"], case["new"], case["batch"], 2)
    return [min(n, c) for n, c in zip(new, ctx)], ctx


def _document_starts(case: dict) -> list[list[int]]:
    """Where the documents of every sequence begin, fixed by the case."""
    out = []
    for b, c in enumerate(_lens(case)[1]):
        r = random.Random(c * 131 + case["documents"] * 7 + b)
        out.append([0] + sorted(r.sample(range(1, c), min(case["documents"], c) - 1)))
    return out


def _sees(case: dict, b: int):
    """(first and end of the tokens at the document's start, first and end of
    the others) that each new token of sequence b attends, numpy [new]."""
    new, ctx = (x[b] for x in _lens(case))
    at = np.arange(ctx - new, ctx)
    starts = np.asarray(_document_starts(case)[b] + [ctx])
    doc = np.searchsorted(starts, at, side="right") - 1
    begin = starts[doc]
    end = np.minimum(starts[doc + 1], np.maximum(at + 1, min(case["prefix"], ctx)))
    first = np.maximum(begin, at - case["window"] + 1) if case["window"] else begin
    kept = np.minimum(begin + (case["sinks"] if case["window"] else 0), first)
    return begin, kept, first, end


def _quotient(a, b):
    """The correctly rounded fp32 quotient of two fp32 tensors."""
    return (a.double() / b.double()).float()


def _encode(x, fmt: str):
    """Codes (int32), fp16 scale and fp16 bias of fp32 rows ``x [..., width]`` in
    groups ``[..., G, group]`` by the format's definition."""
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


def _packed(codes, bits: int):
    """int32 words of codes ``[..., group]``, the first in the lowest bits."""
    per = 32 // bits
    shifts = torch.arange(per, device="cuda", dtype=torch.int64) * bits
    words = (codes.unflatten(-1, (-1, per)).long() << shifts).sum(-1)
    return (words - ((words >> 31) << 32)).int()


def _values(words, scale, bias, fmt: str, width: int):
    """fp32 rows that packed codes, scales and biases stand for."""
    _, bits, _ = _parse(fmt)
    shifts = torch.arange(32 // bits, device="cuda", dtype=torch.int32) * bits
    codes = ((words[..., None] >> shifts) & ((1 << bits) - 1)).flatten(-2)
    if bias is None:
        x = (codes - ((1 << (bits - 1)) - 1)).float() * scale.float()
    else:
        x = codes.float() * scale.float() + bias.float()
    return x.flatten(-2)[..., :width]


def _exact_values(words, scale, bias, fmt: str, width: int):
    """The same in 64 bits, each code cut out of its word."""
    scheme, bits, group = _parse(fmt)
    i = torch.arange(group, device="cuda")
    codes = torch.div((words.long() & 0xFFFFFFFF)[..., i * bits // 32], 2 ** (i * bits % 32), rounding_mode="floor") % 2 ** bits
    x = (codes - (0 if scheme == "a" else 2 ** (bits - 1) - 1)).double() * scale.double()
    return (x if bias is None else x + bias.double()).flatten(-2)[..., :width]


# ---- attend -------------------------------------------------------------------------
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
    codes, scale, bias = _encode(x, fmt)
    held.update(words=_packed(codes, _parse(fmt)[1]), scale=scale, bias=bias)
    at = (tail_at[:, None] + torch.arange(page, device="cuda"))[:, None, :, None].clamp(max=x.shape[2] - 1)
    held["tail"] = torch.gather(x, 2, at.expand(x.shape[0], x.shape[1], page, hd)).half()
    return held


def _held_rows(held: dict):
    """fp32 rows ``[B, H, T, hd]`` of held pages."""
    if held["fmt"] == "m3":
        return held["rows"].float()
    x = _values(held["words"], held["scale"], held["bias"], held["fmt"], held["hd"])
    T, page = x.shape[2], held["page"]
    x = torch.nn.functional.pad(x, (0, 0, 0, page))
    at = (held["tail_at"][:, None] + torch.arange(page, device="cuda"))[:, None, :, None].expand(held["tail"].shape)
    return x.scatter(2, at, held["tail"].float())[:, :, :T]


def _own_filled(case: dict, fmt: str, x, lens, seed: int):
    """A pool that holds rows ``x [B, H, T, hd]``, its pages in any order, and
    the page table ``[B, H, pages]``; the last page of a sequence exact."""
    from dotcache_amd.page_pool import DevicePagePool, PoolGeometry, page_format_of

    B, H, T, hd = x.shape
    P = case["page"]
    W = -(-T // P)
    scheme, bits, group = _parse(fmt)
    pages = B * H * W + B * H
    pool = DevicePagePool(PoolGeometry(hd, group, P), reserve_bytes=pages * P * 2 * hd + (1 << 20), reserve_pages=pages + 16)
    form = page_format_of("M3" if scheme == "m3" else "M0", "symmetric" if scheme == "s" else "affine", bits or 4)
    table = np.random.default_rng(seed).permutation(pool.allocate(*form, B * H * W, tokens=P)).reshape(B, H, W).astype(np.int32)
    last = (np.asarray(lens) - 1) // P
    if fmt != "m3":
        table[np.arange(B), :, last] = pool.allocate(0, 0, B * H, tokens=P).reshape(B, H)
    pool.set_tokens(table[np.arange(B), :, last].ravel(), np.repeat(np.asarray(lens) - last * P, H))
    ids = torch.from_numpy(table).cuda()
    token = torch.arange(T, device="cuda")
    pool.encode_rows(x.reshape(B * H * T, hd), ids[:, :, token // P].reshape(-1).int(),
                     (token % P).int().expand(B, H, T).reshape(-1))
    return pool, ids


def _cache_rows(case: dict, seed: int, tokens: int):
    """Keys and values [B, H, T, hd] that went into the cache: a few channels
    of each head are much larger than the others."""
    out = []
    for tag in (11, 13):
        x = _randn(seed, tag, case["batch"], case["kv_heads"], tokens, case["hd"])
        x = x * torch.exp(0.6 * _randn(seed, tag + 1, 1, case["kv_heads"], 1, case["hd"]))
        out.append(x.to(torch.bfloat16).float())
    return out


def _prepare_attend(case: dict, seed: int) -> dict:
    new, ctx = _lens(case)
    Hq, hd = case["kv_heads"] * case["q_per_kv"], case["hd"]
    rows = _cache_rows(case, seed, max(ctx))
    state = {"case": case, "held": [_pages_of(x, f, case["page"], ctx) for x, f in zip(rows, (case["key"], case["value"]))]}
    state["q"] = _randn(seed, 21, sum(new), Hq, hd).to(_DTYPES[case["dtype"]])
    # (capped scores come from queries that no norm keeps small)
    state["scale"] = (3.0 if case["cap"] else 1.0) / math.sqrt(hd)
    # a slope for every query head, 2^-8 at the least
    state["slopes"] = 2.0 ** (-8.0 * (torch.arange(Hq, device="cuda") + 1) / Hq) if case["slopes"] else None
    # every sequence padded to the longest: which row a padded one repeats, its token, and what it attends
    N = max(new)
    row = np.minimum(np.arange(N), np.asarray(new)[:, None] - 1)
    start = np.concatenate([[0], np.cumsum(new)])[:-1]
    state["from"] = torch.from_numpy(start[:, None] + row).cuda()
    state["to"] = torch.from_numpy(np.concatenate([b * N + np.arange(n) for b, n in enumerate(new)])).cuda()
    state["at"] = torch.from_numpy(np.asarray(ctx)[:, None] - np.asarray(new)[:, None] + row).cuda()
    sees = [np.stack(_sees(case, b), -1)[row[b]] for b in range(case["batch"])]
    state["sees"] = torch.from_numpy(np.stack(sees)).cuda()  # [B, N, 4]
    if own:
        from dotcache_amd.chunk import ChunkMask, plan_chunk

        filled = [_own_filled(case, f, x, ctx, seed + i) for i, (x, f) in enumerate(zip(rows, (case["key"], case["value"])))]
        state["pools"], state["tables"] = zip(*filled)
        mask = ChunkMask(window=case["window"] or None, sinks=case["sinks"] if case["window"] else 0,
                         prefix=[min(case["prefix"], c) for c in ctx] if case["prefix"] else None,
                         documents=_document_starts(case) if case["documents"] > 1 else None)
        state["plan"] = plan_chunk(*state["pools"], new, ctx, kv_heads=case["kv_heads"], q_per_kv=case["q_per_kv"],
                                   dtype=state["q"].dtype, mask=mask)
    return state


def _run_attend(state: dict):
    case = state["case"]
    if own:
        from dotcache_amd.chunk import attend_chunk

        (k_pool, v_pool), (kt, vt) = state["pools"], state["tables"]
        return attend_chunk(k_pool, kt, v_pool, vt, state["q"], state["plan"], query_scale=state["scale"],
                            cap=case["cap"] or None, slopes=state["slopes"])
    H, n_q, hd = case["kv_heads"], case["q_per_kv"], case["hd"]
    k, v = (_held_rows(h) for h in state["held"])
    B, N = state["from"].shape
    q = state["q"][state["from"]].float().reshape(B, N, H, n_q, hd).transpose(1, 2).reshape(B, H, N * n_q, hd)
    s = torch.matmul(q * state["scale"], k.transpose(-1, -2).contiguous()).unflatten(2, (N, n_q))  # [B, H, N, n_q, T]
    if case["cap"]:
        s = torch.tanh_(s.div_(case["cap"])).mul_(case["cap"])
    u = torch.arange(k.shape[2], device="cuda")
    if state["slopes"] is not None:
        away = (state["at"][:, :, None] - u).abs().float()
        for j in range(n_q):
            s[:, :, :, j].sub_(state["slopes"].reshape(H, n_q)[:, j][None, :, None, None] * away[:, None])
    begin, kept, first, end = (x[..., None] for x in state["sees"].unbind(-1))
    seen = ((u >= first) & (u < end)) | ((u >= begin) & (u < kept))
    s = s.masked_fill_(~seen[:, None, :, None], -math.inf).flatten(2, 3)
    p = s.sub_(s.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    o = o.reshape(B, H, N, n_q, hd).transpose(1, 2).reshape(B * N, H * n_q, hd)
    return o[state["to"]].to(state["q"].dtype)


def _exact_held(held: dict, b: int, h: int):
    """One stream's rows in 64 bits."""
    if held["fmt"] == "m3":
        return held["rows"][b, h].double()
    x = _exact_values(held["words"][b, h], held["scale"][b, h], None if held["bias"] is None else held["bias"][b, h],
                      held["fmt"], held["hd"])
    at = int(held["tail_at"][b])
    n = min(held["page"], x.shape[0] - at)
    x[at: at + n] = held["tail"][b, h, :n].double()
    return x


def _exact_attend(case: dict, seed: int):
    s = _prepare_attend(case, seed)
    new, ctx = _lens(case)
    n_q, out, t0 = case["q_per_kv"], torch.empty_like(s["q"], dtype=torch.float64), 0
    for b in range(case["batch"]):
        n, c = new[b], ctx[b]
        i, u = torch.arange(c - n, c, device="cuda")[:, None], torch.arange(c, device="cuda")[None, :]
        starts = torch.zeros(c, dtype=torch.int64, device="cuda")
        starts[torch.tensor(_document_starts(case)[b], device="cuda")] = 1
        doc = starts.cumsum(0)  # which document a token is of
        begins = torch.nonzero(starts).flatten()[doc - 1]
        sees = (doc[i] == doc[u]) & ((u <= i) | (u < case["prefix"]))
        if case["window"]:
            sees &= (i - u < case["window"]) | (u - begins[u] < case["sinks"])
        for h in range(case["kv_heads"]):
            k, v = (_exact_held(x, b, h)[:c] for x in s["held"])
            kt = k.t().contiguous()
            for j in range(h * n_q, (h + 1) * n_q):
                logits = (s["q"][t0: t0 + n, j].double() @ kt) * s["scale"]
                if case["cap"]:
                    e = torch.exp(-2.0 * logits.abs() / case["cap"])
                    logits = torch.sign(logits) * case["cap"] * (1 - e) / (1 + e)
                if case["slopes"]:
                    logits = logits - s["slopes"][j].double() * (i - u).abs()
                w = torch.softmax(torch.where(sees, logits, torch.full_like(logits, -math.inf)), dim=-1)
                out[t0: t0 + n, j] = w @ v
        t0 += n
    return out


# ---- project ------------------------------------------------------------------------
def _prepare_project(case: dict, seed: int) -> dict:
    M, K, N, fmt = case["rows"], case["inputs"], case["outputs"], case["weight"]
    dtype = _DTYPES[case["dtype"]]
    # rows as a norm leaves them, with channels of different sizes; a trained matrix's entries are small
    x = (_randn(seed, 31, M, K) * torch.exp(0.5 * _randn(seed, 32, 1, K))).to(dtype)
    codes, scale, bias = _encode(_randn(seed, 33, N, K) * (0.7 / math.sqrt(K)), fmt)
    state = {"case": case, "x": x, "words": _packed(codes, 4), "scale": scale, "bias": bias}
    if own:
        from dotcache_amd.projection import GroupedWeight

        state["weight"] = GroupedWeight.from_codes(codes.flatten(-2)[:, :K], scale[..., 0],
                                                   None if bias is None else bias[..., 0], group_size=_parse(fmt)[2])
    return state


def _run_project(state: dict):
    if own:
        from dotcache_amd.projection import project

        return project(state["x"], state["weight"])
    case, x = state["case"], state["x"]
    w = _values(state["words"], state["scale"], state["bias"], case["weight"], case["inputs"])
    return torch.matmul(x.float(), w.t()).to(x.dtype)


def _exact_project(case: dict, seed: int):
    s = _prepare_project(case, seed)
    w = _exact_values(s["words"], s["scale"], s["bias"], case["weight"], case["inputs"])
    return s["x"].double() @ w.t().contiguous()


# ---- the interface ------------------------------------------------------------------
def prepare(case: dict, seed: int) -> dict:
    return (_prepare_attend if case["kind"] == "attend" else _prepare_project)(case, seed)


def run(state: dict):
    return (_run_attend if state["case"]["kind"] == "attend" else _run_project)(state)


def exact(case: dict, seed: int):
    return (_exact_attend if case["kind"] == "attend" else _exact_project)(case, seed)


def work(case: dict) -> dict:
    e = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "project":
        M, K, N = case["rows"], case["inputs"], case["outputs"]
        return {"bytes": N * _row_bytes(case["weight"], K) + M * (K + N) * e, "flops": 2 * M * N * K}
    H, hd = case["kv_heads"], case["hd"]
    new, _ = _lens(case)
    pairs = read = 0
    for b in range(case["batch"]):
        begin, kept, first, end = _sees(case, b)
        pairs += int((end - first + kept - begin).sum())
        # tokens that some new token attends
        edges = np.zeros(int(end.max()) + 1, dtype=np.int64)
        for lo, hi in ((begin, kept), (first, end)):
            np.add.at(edges, lo[lo < hi], 1)
            np.add.at(edges, hi[lo < hi], -1)
        read += int((np.cumsum(edges) > 0).sum())
    stored = sum(_row_bytes(case[x], hd) for x in ("key", "value"))
    return {"bytes": H * (read * stored + 2 * sum(new) * case["q_per_kv"] * hd * e), "flops": 4 * pairs * H * case["q_per_kv"] * hd}
