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

The plan depends on the lengths alone, so that one plan serves every layer of a
step.  The reference decodes one token at a time (reference
``dotcache/integrations/llama.py:424-425``).
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


def _torch():
    import torch

    return torch


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
               dtype=None, target_items: int | None = None) -> ChunkPlan:
    """The plan for ``new[b]`` new tokens (0: a sequence that waits) of
    ``context[b]`` tokens in all, on the pools' device.  ``dtype``, the
    queries' type, is checked if given; a plan serves any of them."""
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
    L = _lib.lib()
    counts = [C.c_int32() for _ in range(5)]  # items, few, few rows, merges, partial rows

    def plan(items, merges):
        return L.dc_plan_chunk(n.ctypes.data, ctx.ctypes.data, n.size, int(kv_heads), int(q_per_kv), pool.geometry.head_dim,
                               target, MIN_SPLIT_TOKENS, items.ctypes.data, items.shape[0], *(C.byref(c) for c in counts[:3]),
                               merges.ctypes.data, merges.shape[0], *(C.byref(c) for c in counts[3:]))

    empty = [np.zeros((0, len(f)), dtype=np.int32) for f in (_lib.CHUNK_ITEM_FIELDS, _lib.CHUNK_MERGE_FIELDS)]
    st = plan(*empty)
    if st != _lib.DC_ESPACE:
        _lib.check(st, "dc_plan_chunk")
    items, merges = (np.zeros((c.value, e.shape[1]), dtype=np.int32) for c, e in zip((counts[0], counts[3]), empty))
    _lib.check(plan(items, merges), "dc_plan_chunk")
    both = torch.from_numpy(np.concatenate([items.ravel(), merges.ravel()])).to(pool.arena.device)
    busy = ctx[n > 0]
    return ChunkPlan(items=both[: items.size].view(items.shape), merges=both[items.size:].view(merges.shape),
                     n_items=items.shape[0], n_few=counts[1].value, few_rows=counts[2].value, n_merges=merges.shape[0],
                     n_partials=counts[4].value, host_items=items, host_merges=merges,
                     new=n, context=ctx, kv_heads=int(kv_heads), q_per_kv=int(q_per_kv),
                     n_tokens=int(n.sum(dtype=np.int64)), max_context=int(busy.max()) if busy.size else 0)


def _check_pools(pool: DevicePagePool, vpool: DevicePagePool) -> None:
    g = pool.geometry
    if (vpool.geometry.head_dim, vpool.geometry.page_capacity) != (g.head_dim, g.page_capacity):
        raise ValueError("key and value pools must share head_dim and page_capacity")
    if vpool.arena.device != pool.arena.device:
        raise ValueError("key and value pools must be on one device")
    if g.head_dim > MAX_HEAD_DIM:
        raise ValueError(f"chunk attention takes head_dim up to {MAX_HEAD_DIM}")


def workspace_bytes(plan: ChunkPlan, head_dim: int) -> int:
    return int(_lib.lib().dc_chunk_workspace_bytes(plan.n_partials, int(head_dim)))


def attend_chunk(pool: DevicePagePool, k_table, v_pool: DevicePagePool | None, v_table, queries, plan: ChunkPlan, *,
                 query_scale: float = 1.0, out=None, workspace=None, validate: bool = False):
    """Causal attention of ``queries [tokens, Hq, head_dim]`` (fp32, fp16 or
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
    may have either sign, or be 0.  ``workspace``: uint8, :func:`workspace_bytes`
    at least, 16-byte aligned, not shared by calls that may overlap (default: one
    of its own).  ``validate`` reads the tables back and checks them against the
    pools (the kernel itself leaves out, and never reads, what a table does not
    name).

    The kernel follows from the formats that the pools have ever held.  Once a
    pool has taken a 2- or 3-bit, int8 or fp32 page (a cache's tail, by
    ``escape_dtype``), 16-bit queries take the general kernel, two to six times
    as long; and a captured call is captured anew once a pool takes pages of a
    format that it had not."""
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
        out = torch.empty(queries.shape, dtype=queries.dtype, device=device)
    elif out.shape != queries.shape or out.dtype != queries.dtype:
        raise ValueError("out must have the queries' shape and dtype")
    q_rows, out_rows = token_rows(queries, "queries", hd, device), token_rows(out, "out", hd, device)
    if validate:
        _validate(pool, vpool, k_table, v_table, plan)
    need = workspace_bytes(plan, hd)
    if need == 0:
        workspace = None
    elif workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    elif workspace.numel() * workspace.element_size() < need or not workspace.is_contiguous() or workspace.device != device:
        raise ValueError(f"workspace must be contiguous, {need} bytes at least, on {device}")
    elif workspace.data_ptr() % 16:
        raise ValueError("workspace must be 16-byte aligned")
    if plan.n_items:
        call_on(device, _lib.lib().dc_attend_chunk, "dc_attend_chunk", pool.c_pool(), vpool.c_pool(), k_table.data_ptr(),
                v_table.data_ptr(), shape[2], plan.items.data_ptr(), plan.n_items, plan.n_few, plan.few_rows,
                plan.merges.data_ptr(), plan.n_merges, plan.n_partials, B, plan.kv_heads, plan.n_tokens, q_rows, float(query_scale), out_rows,
                workspace.data_ptr() if need else None, need)
    return out


def attend_cached(cache, queries, new: np.ndarray, context: np.ndarray, k_table, v_table, q_head_to_kv_head, default_map,
                  query_scale: float):
    """:func:`attend_chunk` of ``queries [tokens, Hq, hd]`` over a cache's pages,
    its query heads in any order (``q_head_to_kv_head``; None: ``default_map``).
    ``cache`` keeps the last plan, by its lengths (every layer of a step has the
    same) and the stream it was made on, whose order its memory's reuse follows;
    each call has a workspace of its own.  A captured call would read the plan
    after the cache has dropped it, so it is refused."""
    torch = _torch()
    if queries.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("a cache's chunk attention cannot be captured: capture attend_chunk with a plan of your own")
    H = cache.num_key_value_heads
    Hq = cache.num_attention_heads
    qmap = default_map if q_head_to_kv_head is None else np.asarray(q_head_to_kv_head, dtype=np.int64)
    if qmap.shape != (Hq,) or np.any(qmap < 0) or np.any(qmap >= H) or np.any(np.bincount(qmap, minlength=H) != Hq // H):
        raise ValueError("q_head_to_kv_head must give every KV head the same number of query heads")
    key = (new.tobytes(), context.tobytes(), torch.cuda.current_stream(queries.device).cuda_stream if queries.is_cuda else 0)
    if cache._chunk_plan is None or cache._chunk_plan[0] != key:
        cache._chunk_plan = (key, plan_chunk(cache.k_pool, cache.v_pool, new, context, kv_heads=H, q_per_kv=Hq // H))
    plan = cache._chunk_plan[1]
    order = np.argsort(qmap, kind="stable")  # query heads grouped by KV head
    if np.array_equal(order, np.arange(Hq)):
        return attend_chunk(cache.k_pool, k_table, cache.v_pool, v_table, queries, plan, query_scale=query_scale)
    at = torch.from_numpy(order).to(cache.device)
    out = attend_chunk(cache.k_pool, k_table, cache.v_pool, v_table, queries[:, at], plan, query_scale=query_scale)
    res = torch.empty_like(out)
    res[:, at] = out
    return res


def _validate(pool: DevicePagePool, vpool: DevicePagePool, k_table, v_table, plan: ChunkPlan) -> None:
    """ValueError unless every sequence with new tokens has the live pages its
    context needs, each full but the last."""
    P = pool.geometry.page_capacity
    kt, vt = k_table.cpu().numpy(), v_table.cpu().numpy()
    for b in np.flatnonzero(plan.new > 0).tolist():
        pages = -(-int(plan.context[b]) // P)
        want = np.full(pages, P, dtype=np.int64)
        want[-1] = plan.context[b] - (pages - 1) * P
        for p, t in ((pool, kt), (vpool, vt)):
            ids = t[b, :, :pages]
            p.validate_ids(ids)
            if np.any(p.tokens_of(ids) != want):
                raise ValueError(f"sequence {b}: its pages do not hold a context of {int(plan.context[b])} tokens")


__all__ = ["ChunkPlan", "attend_chunk", "plan_chunk", "workspace_bytes"]
