"""Attention of a chunk of new tokens over paged sequences
(``dc_attend_chunk``): a prompt's chunks, drafted tokens to verify and plain
decodes of one batch in one call, causal among the new tokens.

The counterpart of :func:`~dotcache_amd.decode.decode_paged` for more than one
query token per sequence: same pools, same page tables, any page format.
Sequence b has ``new[b]`` new tokens of a context of ``context[b]`` tokens with
them; its new tokens' keys and values are in its pages already (append first),
and new token i attends tokens ``0 .. context[b] - new[b] + i``.  The queries
of all sequences lie one after another in one tensor.  Every page of a
sequence but the last is full, as the caches keep them.

The plan depends on the lengths and the mask alone, so that one plan serves
every layer of a step that has that mask.  The reference decodes one token at a
time (reference ``dotcache/integrations/llama.py:424-425``).

Which tokens a new token attends may be narrowed or widened by a
:class:`ChunkMask` (a sliding window, a prefix, documents), and scores may be
capped by a tanh and lowered by the distance (``cap``, ``slopes``):

    s = query_scale q . k;   s = cap tanh(s / cap);   s -= slope |i - u|

for token i and the token u that it attends, slopes by query head.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import numpy as np

from . import _lib
from .decode import default_target_items
from .page_pool import DevicePagePool, call_on
from .rotary import token_rows

MAX_HEAD_DIM = 256
# A token range that a tile of query rows is split into holds at least this
# many tokens.
MIN_SPLIT_TOKENS = 128
MAX_PLANS = 8  # masks for which a cache keeps the plan of a step


def _torch():
    import torch

    return torch


def _whole(x, name: str, least: int) -> int:
    if not isinstance(x, (int, np.integer)) or isinstance(x, bool) or not least <= x < 2 ** 31:
        raise ValueError(f"{name} must be an integer from {least} on")
    return int(x)


@dataclass(frozen=True)
class ChunkMask:
    """Which tokens of its sequence a token i attends: those u that are not
    behind it (u <= i), or in the sequence's first ``prefix`` tokens with it,

    * of its own document (``documents``: for each sequence where its documents
      begin, ascending from 0; None: one document each),
    * not ``window`` tokens or more ahead of it (u > i - window: up to itself the
      last ``window``), or among its document's first ``sinks`` (None: no window).

    ``prefix`` is a number for all sequences or one for each; its tokens see
    each other both ways (those behind a token at any distance, a window or not),
    so a chunk that ends inside it belongs to no complete prompt and is refused.
    Equal masks compare equal."""
    window: int | None = None
    sinks: int = 0
    prefix: int | tuple | None = None
    documents: tuple | None = None

    def __post_init__(self):
        put = lambda name, x: object.__setattr__(self, name, x)  # noqa: E731
        if self.window is not None:
            put("window", _whole(self.window, "window", 1))
        put("sinks", _whole(self.sinks, "sinks", 0))
        if self.sinks and self.window is None:
            raise ValueError("sinks are what a window leaves in sight: they need a window")
        if self.prefix is not None:
            x = self.prefix.tolist() if hasattr(self.prefix, "tolist") else self.prefix
            put("prefix", tuple(_whole(y, "prefix", 0) for y in x) if isinstance(x, (list, tuple)) else _whole(x, "prefix", 0))
        if self.documents is not None:
            rows = []
            for starts in self.documents:
                starts = tuple(_whole(y, "a document's start", 0) for y in (starts.tolist() if hasattr(starts, "tolist") else starts))
                if starts and (starts[0] != 0 or any(y <= x for x, y in zip(starts, starts[1:]))):
                    raise ValueError("documents must begin at ascending tokens, the first at 0")
                rows.append(starts)
            put("documents", tuple(rows))

    def ranges(self, new, context) -> np.ndarray:
        """int32 ``[tokens, 4]``: new token t attends tokens ``r[0] .. r[1] - 1``
        (the sinks) and ``r[2] .. r[3] - 1`` of its sequence."""
        new, ctx = _lengths(new, "new").astype(np.int64), _lengths(context, "context").astype(np.int64)
        if new.shape != ctx.shape or np.any(new > ctx):
            raise ValueError("context must hold one length per sequence, with its new tokens")
        seq = np.repeat(np.arange(new.size), new)
        at = np.arange(int(new.sum())) - np.repeat(np.cumsum(new) - new, new) + (ctx - new)[seq]
        begin, stop = np.zeros_like(at), ctx[seq]
        if self.documents is not None:
            if len(self.documents) != new.size:
                raise ValueError("documents must hold one list of starts per sequence")
            t = 0
            for b, starts in enumerate(self.documents):
                if starts and starts[-1] >= max(int(ctx[b]), 1):
                    raise ValueError(f"sequence {b}: a document begins past its context")
                edges = np.asarray((starts or (0,)) + (int(ctx[b]),))
                n = int(new[b])
                doc = np.searchsorted(edges[:-1], at[t: t + n], side="right")
                begin[t: t + n], stop[t: t + n] = edges[doc - 1], edges[doc]
                t += n
        end = at + 1
        if self.prefix is not None:
            prefix = np.asarray(self.prefix, dtype=np.int64)
            if prefix.ndim and prefix.shape != new.shape:
                raise ValueError("prefix must be a number, or hold one per sequence")
            prefix = np.broadcast_to(prefix, new.shape)
            if np.any((prefix > ctx) & (new > 0)):
                raise ValueError("a prefix must lie in its sequence's context")
            end = np.minimum(np.maximum(end, prefix[seq]), stop)
        first = begin if self.window is None else np.maximum(begin, at - self.window + 1)
        return np.stack([begin, np.minimum(begin + self.sinks, first), first, end], axis=1).astype(np.int32)


@dataclass
class ChunkPlan:
    """Work of one :func:`attend_chunk` call (:func:`plan_chunk`)."""
    items: object            # device int32 [n_items, 9]: dc_chunk_item
    merges: object           # device int32 [n_merges, 6]: dc_chunk_merge
    n_items: int
    n_few: int               # the first of them: sequences of few rows, at most few_rows each
    few_rows: int
    n_merges: int
    n_partials: int          # rows of partial results
    host_items: np.ndarray
    host_merges: np.ndarray
    new: np.ndarray          # new tokens of every sequence
    context: np.ndarray      # tokens of every sequence, with the new ones
    kv_heads: int
    q_per_kv: int
    n_tokens: int            # query rows [n_tokens, kv_heads * q_per_kv, head_dim]
    max_context: int         # of the sequences that have new tokens
    ranges: object = None    # with a mask: device int32 [n_tokens, 4], what each new token attends ...
    gaps: object = None      # ... and [n_items, 2], tokens that an item leaves out
    host_ranges: np.ndarray | None = None
    host_gaps: np.ndarray | None = None


def _lengths(x, name: str) -> np.ndarray:
    if hasattr(x, "detach"):
        x = x.detach().cpu().numpy()
    x = np.asarray(x)
    if x.ndim != 1 or x.size == 0 or not np.issubdtype(x.dtype, np.integer):
        raise ValueError(f"{name} must hold one integer per sequence")
    if x.min() < 0 or x.max() >= 2 ** 31:
        raise ValueError(f"{name} must lie in [0, 2^31)")
    return np.ascontiguousarray(x, dtype=np.int32)


def plan_chunk(pool: DevicePagePool, v_pool: DevicePagePool | None, new, context, *, kv_heads: int, q_per_kv: int,
               dtype=None, target_items: int | None = None, mask=None) -> ChunkPlan:
    """The plan for ``new[b]`` new tokens (0: a sequence that waits) of
    ``context[b]`` tokens in all, on the pools' device.  ``dtype``, the
    queries' type, is checked if given; a plan serves any of them.

    ``mask``: a :class:`ChunkMask` (None: causal), or int32 ``[tokens, 4]``
    for a mask of another kind: new token t attends tokens ``mask[t, 0] ..
    mask[t, 1] - 1`` and ``mask[t, 2] .. mask[t, 3] - 1`` of its sequence (once
    each, where the two overlap), empty ranges where begin and end are equal; a
    token that attends none gets zeros."""
    torch = _torch()
    vpool = pool if v_pool is None else v_pool
    _check_pools(pool, vpool)
    n, ctx = _lengths(new, "new"), _lengths(context, "context")
    if n.shape != ctx.shape:
        raise ValueError("new and context must hold one length per sequence")
    if np.any(n > ctx):
        raise ValueError("a sequence's context includes its new tokens")
    if dtype is not None and dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise ValueError(f"unsupported query dtype {dtype}")
    if int(kv_heads) <= 0 or int(q_per_kv) <= 0:
        raise ValueError("kv_heads and q_per_kv must be positive")
    target = default_target_items() // 4 if target_items is None else int(target_items)
    if target <= 0:
        raise ValueError("target_items must be positive")
    ranges = None
    if isinstance(mask, ChunkMask):
        ranges = mask.ranges(n, ctx) if mask != ChunkMask() else None
    elif mask is not None:
        ranges = np.asarray(mask.detach().cpu().numpy() if hasattr(mask, "detach") else mask)
        if ranges.shape != (int(n.sum(dtype=np.int64)), 4) or not np.issubdtype(ranges.dtype, np.integer):
            raise ValueError("mask must be a ChunkMask, or integers of shape [new tokens, 4]")
        if ranges.size and (ranges.min() < 0 or ranges.max() >= 2 ** 31):
            raise ValueError("mask has a range outside its context")
        ranges = np.ascontiguousarray(ranges, dtype=np.int32)
    L = _lib.lib()
    counts = [C.c_int32() for _ in range(5)]  # items, few, few rows, merges, partial rows

    def plan(items, merges, gaps):
        shape = (n.size, int(kv_heads), int(q_per_kv), pool.geometry.head_dim, target, MIN_SPLIT_TOKENS)
        tail = (items.shape[0], *(C.byref(c) for c in counts[:3]), merges.ctypes.data, merges.shape[0],
                *(C.byref(c) for c in counts[3:]))
        if ranges is None:
            return L.dc_plan_chunk(n.ctypes.data, ctx.ctypes.data, *shape, items.ctypes.data, *tail)
        return L.dc_plan_chunk_ranges(n.ctypes.data, ctx.ctypes.data, ranges.ctypes.data, *shape, items.ctypes.data,
                                      gaps.ctypes.data, *tail)

    what = "dc_plan_chunk" if ranges is None else "dc_plan_chunk_ranges"
    empty = [np.zeros((0, len(f)), dtype=np.int32) for f in (_lib.CHUNK_ITEM_FIELDS, _lib.CHUNK_MERGE_FIELDS, "gg")]
    st = plan(*empty)
    if st != _lib.DC_ESPACE:
        _lib.check(st, what)
    items, merges, gaps = (np.zeros((c.value, e.shape[1]), dtype=np.int32) for c, e in zip((counts[0], counts[3], counts[0]), empty))
    _lib.check(plan(items, merges, gaps), what)
    # (ranges and gaps first, at multiples of 16 and 8 bytes)
    parts = [items, merges] if ranges is None else [ranges, gaps, items, merges]
    both = torch.from_numpy(np.concatenate([x.ravel() for x in parts])).to(pool.arena.device)
    *masked, items_d, merges_d = (d.view(x.shape) for d, x in zip(both.split([x.size for x in parts]), parts))
    busy = ctx[n > 0]
    return ChunkPlan(items=items_d, merges=merges_d, n_items=items.shape[0], n_few=counts[1].value, few_rows=counts[2].value, n_merges=merges.shape[0],
                     n_partials=counts[4].value, host_items=items, host_merges=merges,
                     new=n, context=ctx, kv_heads=int(kv_heads), q_per_kv=int(q_per_kv),
                     n_tokens=int(n.sum(dtype=np.int64)), max_context=int(busy.max()) if busy.size else 0,
                     ranges=masked[0] if masked else None, gaps=masked[1] if masked else None, host_ranges=ranges,
                     host_gaps=gaps if masked else None)


def _check_pools(pool: DevicePagePool, vpool: DevicePagePool) -> None:
    g = pool.geometry
    if (vpool.geometry.head_dim, vpool.geometry.page_capacity) != (g.head_dim, g.page_capacity):
        raise ValueError("key and value pools must share head_dim and page_capacity")
    if vpool.arena.device != pool.arena.device:
        raise ValueError("key and value pools must be on one device")
    if g.head_dim > MAX_HEAD_DIM:
        raise ValueError(f"chunk attention takes head_dim up to {MAX_HEAD_DIM}")


def _check_slopes(slopes, heads: int, device) -> None:
    if slopes is not None and (not isinstance(slopes, _torch().Tensor) or slopes.shape != (heads,) or slopes.dtype != _torch().float32
                               or slopes.device != device or not slopes.is_contiguous()):
        raise ValueError(f"slopes must be contiguous fp32 [{heads}] on {device}")


def workspace_bytes(plan: ChunkPlan, head_dim: int) -> int:
    return int(_lib.lib().dc_chunk_workspace_bytes(plan.n_partials, int(head_dim)))


def attend_chunk(pool: DevicePagePool, k_table, v_pool: DevicePagePool | None, v_table, queries, plan: ChunkPlan, *,
                 query_scale: float = 1.0, cap: float | None = None, slopes=None, out=None, workspace=None,
                 validate: bool = False):
    """Attention (causal, or by the plan's mask) of ``queries [tokens, Hq, head_dim]`` (fp32, fp16 or
    bf16, any token and head stride) over the pages that ``k_table`` /
    ``v_table`` (int32 device ``[n_seqs, kv_heads, pages]``) name in ``pool`` /
    ``v_pool`` (None: the same pool); query head h reads KV head ``h //
    q_per_kv``.  Returns rows of the queries' shape and type (or writes
    ``out``: same shape and type, apart from the queries; rows past the plan's
    tokens are left as they are).

    With 16-bit queries, the queries, the pages' values and the softmax weights
    are fp16 matrix operands, each rounded once, and all sums fp32: an output is
    off by about 2^-11 of its terms, beside its own rounding.  Values past
    +-65504 overflow, as in fp16 pages; bf16 queries below 2^-14 lose bits, below
    2^-25 they are zeros.  With fp32 queries everything is fp32.  ``query_scale``
    may have either sign, or be 0.  ``cap`` (positive; None: none) and ``slopes``
    (fp32 device ``[Hq]``, any sign; None: none) shape the scores in fp32, in that
    order, before the mask; a capped score is off by about 2^-21 of itself, or,
    with 16-bit queries and a cap up to 256, of the cap.  No gradient flows through
    the call.  ``workspace``: uint8, :func:`workspace_bytes` at least, 16-byte
    aligned, not shared by calls that may overlap (default: one of its own).  ``validate`` reads the tables back and checks them against the
    pools (the kernel itself leaves out, and never reads, what a table does not
    name).

    The kernel follows from the formats that the pools have ever held.  Once a
    pool has taken a 2- or 3-bit, int8 or fp32 page (a cache's tail, by
    ``escape_dtype``), 16-bit queries take the general kernel, two to six times
    as long (decodes of long contexts at head_dim 256: fifteen times); and a
    captured call is captured anew once a pool takes pages of a format that it
    had not."""
    torch = _torch()
    vpool = pool if v_pool is None else v_pool
    _check_pools(pool, vpool)
    hd, P, device = pool.geometry.head_dim, pool.geometry.page_capacity, pool.arena.device
    B = plan.new.size
    shape = tuple(k_table.shape)
    if k_table.dim() != 3 or shape[:2] != (B, plan.kv_heads) or tuple(v_table.shape) != shape:
        raise ValueError(f"page tables must have shape [{B}, {plan.kv_heads}, pages]")
    if k_table.dtype != torch.int32 or v_table.dtype != torch.int32 or not (k_table.is_contiguous() and v_table.is_contiguous()):
        raise ValueError("page tables must be contiguous int32")
    if k_table.device != device or v_table.device != device or plan.items.device != device:
        raise ValueError(f"tables and plan must be on {device}")
    if shape[2] * P < plan.max_context:
        raise ValueError("a context needs more pages than its page-table row holds")
    if queries.dim() != 3 or queries.shape[0] < plan.n_tokens or queries.shape[1] != plan.kv_heads * plan.q_per_kv:
        raise ValueError(f"queries must have shape [{plan.n_tokens}, {plan.kv_heads * plan.q_per_kv}, {hd}]")
    if out is None:
        if queries.shape[0] != plan.n_tokens:
            raise ValueError("queries past the plan's tokens (padding) need an out tensor, whose rows there are left")
        out = queries.new_empty(queries.shape)
    elif out.shape != queries.shape or out.dtype != queries.dtype:
        raise ValueError("out must have the queries' shape and dtype")
    q_rows, out_rows = token_rows(queries, "queries", hd, device), token_rows(out, "out", hd, device)
    if cap is not None and not (0.0 < C.c_float(cap).value < float("inf")):
        raise ValueError("cap must be positive in fp32, or None for none")
    _check_slopes(slopes, queries.shape[1], device)
    if validate:
        _validate(pool, vpool, k_table, v_table, plan)
    need = workspace_bytes(plan, hd)
    if need == 0:
        workspace = None
    elif workspace is None:
        workspace = queries.new_empty(need, dtype=torch.uint8)
    elif workspace.numel() * workspace.element_size() < need or not workspace.is_contiguous() or workspace.device != device:
        raise ValueError(f"workspace must be contiguous, {need} bytes at least, on {device}")
    elif workspace.data_ptr() % 16:
        raise ValueError("workspace must be 16-byte aligned")
    if plan.n_items:
        args = (pool.c_pool(), vpool.c_pool(), k_table.data_ptr(), v_table.data_ptr(), shape[2], plan.items.data_ptr(), plan.n_items,
                plan.n_few, plan.few_rows, plan.merges.data_ptr(), plan.n_merges, plan.n_partials, B, plan.kv_heads, plan.n_tokens,
                q_rows, float(query_scale))
        tail = (out_rows, workspace.data_ptr() if need else None, need)
        if cap is None and slopes is None and plan.ranges is None:
            call_on(device, _lib.lib().dc_attend_chunk, "dc_attend_chunk", *args, *tail)
        else:
            rule = _lib.ScoreRule(0.0 if cap is None else float(cap), None if slopes is None else slopes.data_ptr(),
                                  None if plan.ranges is None else plan.ranges.data_ptr(),
                                  None if plan.gaps is None else plan.gaps.data_ptr())
            call_on(device, _lib.lib().dc_attend_chunk_rule, "dc_attend_chunk_rule", *args, rule, *tail)
    return out


def attend_cached(cache, queries, new: np.ndarray, context: np.ndarray, k_table, v_table, q_head_to_kv_head, default_map,
                  query_scale: float, mask=None, cap=None, slopes=None):
    """:func:`attend_chunk` of ``queries [tokens, Hq, hd]`` over a cache's pages,
    its query heads in any order (``q_head_to_kv_head``; None: ``default_map``).
    ``cache`` keeps the last plans, by their lengths (every layer of a step has
    the same), the stream they were made on, whose order their memory's reuse
    follows, and the masks of the step's layers (:class:`ChunkMask` or None); each call has a workspace of its own.  A captured call would read the plan
    after the cache has dropped it, so it is refused."""
    torch = _torch()
    if queries.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("a cache's chunk attention cannot be captured: capture attend_chunk with a plan of your own")
    H = cache.num_key_value_heads
    Hq = cache.num_attention_heads
    qmap = default_map if q_head_to_kv_head is None else np.asarray(q_head_to_kv_head, dtype=np.int64)
    if qmap.shape != (Hq,) or np.any(qmap < 0) or np.any(qmap >= H) or np.any(np.bincount(qmap, minlength=H) != Hq // H):
        raise ValueError("q_head_to_kv_head must give every KV head the same number of query heads")
    if mask is not None and not isinstance(mask, ChunkMask):
        raise ValueError("a cache's mask must be a ChunkMask")
    _check_slopes(slopes, Hq, cache.k_pool.arena.device)  # (ahead of their reordering)
    key = (new.tobytes(), context.tobytes(), torch.cuda.current_stream(queries.device).cuda_stream if queries.is_cuda else 0)
    if cache._chunk_plan is None or cache._chunk_plan[0] != key:
        cache._chunk_plan = (key, {})
    plans = cache._chunk_plan[1]
    if mask not in plans:
        if len(plans) >= MAX_PLANS:
            plans.clear()
        plans[mask] = plan_chunk(cache.k_pool, cache.v_pool, new, context, kv_heads=H, q_per_kv=Hq // H, mask=mask)
    plan = plans[mask]
    order = np.argsort(qmap, kind="stable")  # query heads grouped by KV head
    if np.array_equal(order, np.arange(Hq)):
        return attend_chunk(cache.k_pool, k_table, cache.v_pool, v_table, queries, plan, query_scale=query_scale, cap=cap,
                            slopes=slopes)
    at = torch.from_numpy(order).to(cache.device)
    out = attend_chunk(cache.k_pool, k_table, cache.v_pool, v_table, queries[:, at], plan, query_scale=query_scale, cap=cap,
                       slopes=None if slopes is None else slopes[at])
    res = torch.empty_like(out)
    res[:, at] = out
    return res


def _validate(pool: DevicePagePool, vpool: DevicePagePool, k_table, v_table, plan: ChunkPlan) -> None:
    """ValueError unless every sequence with new tokens has the live pages its
    context needs (with a mask: those with a token that a new one attends),
    each full but the last."""
    P = pool.geometry.page_capacity
    kt, vt = k_table.cpu().numpy(), v_table.cpu().numpy()
    start = np.cumsum(plan.new, dtype=np.int64) - plan.new
    for b in np.flatnonzero(plan.new > 0).tolist():
        pages = -(-int(plan.context[b]) // P)
        want = np.full(pages, P, dtype=np.int64)
        want[-1] = plan.context[b] - (pages - 1) * P
        need = np.ones(pages, dtype=bool)
        if plan.host_ranges is not None:
            r = plan.host_ranges[start[b]: start[b] + plan.new[b]]
            edges = np.zeros(pages + 1, dtype=np.int64)
            for lo, hi in ((r[:, 0], r[:, 1]), (r[:, 2], r[:, 3])):
                np.add.at(edges, lo[lo < hi] // P, 1)
                np.add.at(edges, (hi[lo < hi] - 1) // P + 1, -1)
            need = np.cumsum(edges[:-1]) > 0
        for p, t in ((pool, kt), (vpool, vt)):
            ids = t[b, :, :pages][:, need]
            p.validate_ids(ids)
            if np.any(p.tokens_of(ids) != want[need]):
                raise ValueError(f"sequence {b}: its pages do not hold a context of {int(plan.context[b])} tokens")


__all__ = ["ChunkMask", "ChunkPlan", "attend_chunk", "plan_chunk", "workspace_bytes"]
