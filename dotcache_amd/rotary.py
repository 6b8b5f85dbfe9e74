"""Per-head norms and the position rotation of new queries and keys
(``dc_norm_rotate``), the step between a layer's projections and its cache.

    y = x / sqrt(mean(x^2) + eps) * weight             (per head; weight optional)
    z_a = y_a cos - y_b sin,   z_b = y_b cos + y_a sin

for the pairs (a, b) = (i, i + rotary_dim / 2), or (2 i, 2 i + 1) interleaved;
channels past ``rotary_dim`` are only normed.  The reference's model wrappers
do this in their models (reference ``dotcache/integrations/llama.py:345-358``)
and hand the rows to the cache; here it is one launch, or part of the launch
that writes the pages (:meth:`~dotcache_amd.page_pool.DevicePagePool.append_rotary_with`).

Rows are token-major ``[tokens, heads, head_dim]`` in fp32, fp16 or bf16 with
any token and head stride, so queries, keys and values may be views of one
projection's output.  Sums and products are fp32 (fp64 for keys on their way
into pages), rounded once to the output's type.
"""
from __future__ import annotations

import numpy as np

from . import _lib
from .page_pool import call_on, dtype_code

_NO_ROWS = _lib.TokenRows()
_NO_NORM = _lib.Norm()
_NO_ROTARY = _lib.Rotary()
_ABSENT = (_NO_ROWS, _NO_NORM, _NO_ROWS)


def _torch():
    import torch

    return torch


class RotaryTable:
    """Cosines and sines of positions ``[0, n_positions)``, computed in fp64
    (a far position's angle loses its fraction in fp32) and kept in fp32 on
    the device: ``table [n_positions, rotary_dim]``, a position's cosines and
    then its sines.

    ``rotary_dim`` (default ``head_dim``, even) channels are rotated, in pairs
    split by halves or, ``interleaved``, in neighbouring pairs.  ``inv_freq``
    gives ``rotary_dim / 2`` angles per position (default ``base ** (-2 i /
    rotary_dim)``); ``amplitude`` scales the table, as context-extension
    schemes ask for.
    """

    def __init__(self, head_dim: int, n_positions: int, *, rotary_dim: int | None = None, base: float = 10000.0,
                 inv_freq=None, interleaved: bool = False, amplitude: float = 1.0, device="cuda"):
        torch = _torch()
        rd = int(head_dim) if rotary_dim is None else int(rotary_dim)
        if rd <= 0 or rd > int(head_dim) or rd % 2:
            raise ValueError("rotary_dim must be even and in [2, head_dim]")
        if not 0 < int(n_positions) < 2 ** 31:
            raise ValueError("n_positions must be positive")
        freq = float(base) ** (-np.arange(0, rd, 2, dtype=np.float64) / rd) if inv_freq is None else inv_freq
        freq = torch.as_tensor(np.asarray(freq.cpu() if isinstance(freq, torch.Tensor) else freq, dtype=np.float64))
        if tuple(freq.shape) != (rd // 2,):
            raise ValueError(f"inv_freq must hold {rd // 2} frequencies")
        self.head_dim, self.rotary_dim, self.interleaved = int(head_dim), rd, bool(interleaved)
        self.n_positions = int(n_positions)
        angle = torch.arange(self.n_positions, dtype=torch.float64, device=device)[:, None] * freq.to(device)
        self.table = torch.cat([angle.cos() * float(amplitude), angle.sin() * float(amplitude)], dim=-1).float()
        self._c = _lib.Rotary(self.table.data_ptr(), self.n_positions, rd, int(self.interleaved))


def token_rows(x, name: str, head_dim: int, device) -> _lib.TokenRows:
    """``dc_token_rows`` of a tensor ``[tokens, heads, head_dim]``."""
    shape, stride = x.shape, x.stride()
    if len(shape) != 3 or shape[2] != head_dim or (stride[2] != 1 and head_dim > 1):
        raise ValueError(f"{name} must have shape [tokens, heads, {head_dim}] with contiguous channels")
    if x.device != device:
        raise ValueError(f"{name} must be on {device}")
    if shape[1] == 0:
        raise ValueError(f"{name} must have at least one head")
    return _lib.TokenRows(x.data_ptr(), stride[0], stride[1], shape[1], dtype_code(x))


def head_norm(weight, name: str, heads: int, head_dim: int, eps: float, device) -> _lib.Norm:
    """``dc_norm`` of a weight ``[head_dim]`` or ``[heads, head_dim]`` (None: no norm)."""
    if weight is None:
        return _NO_NORM
    shape = weight.shape
    if (shape != (head_dim,) and shape != (heads, head_dim)) or not weight.is_contiguous():
        raise ValueError(f"{name} must be contiguous, [{head_dim}] or [{heads}, {head_dim}]")
    if weight.device != device:
        raise ValueError(f"{name} must be on {device}")
    if not eps >= 0.0:
        raise ValueError("eps must be non-negative")
    return _lib.Norm(weight.data_ptr(), dtype_code(weight), head_dim if len(shape) == 2 else 0, eps)


def index_tensor(x, name: str, tokens: int, device, limit: int | None = None):
    """``x`` as a contiguous int32 device tensor of one entry per token.
    Host values (a list or numpy array) are checked against ``[0, limit)``;
    device values are guarded by the kernels."""
    torch = _torch()
    if type(x) is torch.Tensor and x.dtype is torch.int32 and x.shape == (tokens,) and x.device == device and x.is_contiguous() \
            and device.type != "cpu":
        return x
    if not isinstance(x, torch.Tensor) or x.device.type == "cpu":
        host = np.asarray(x)
        if host.size and not np.issubdtype(host.dtype, np.integer):
            raise ValueError(f"{name} must hold integers")
        if limit is not None and host.size and (host.min() < 0 or host.max() >= limit):
            raise ValueError(f"{name} must lie in [0, {limit})")
        if host.size and (host.min() < -2 ** 31 or host.max() >= 2 ** 31):
            raise ValueError(f"{name} must be 32-bit integers")
        x = torch.from_numpy(np.ascontiguousarray(host.astype(np.int32))).to(device)
    if x.dim() != 1 or x.shape[0] != tokens:
        raise ValueError(f"{name} must have one entry per token")
    if x.device != device:
        raise ValueError(f"{name} must be on {device}")
    if x.dtype != torch.int32:
        if x.dtype != torch.int64:
            raise ValueError(f"{name} must be int32 or int64")
        # (values past 32 bits saturate, so that they stay outside every table)
        x = x.clamp(-1, 2 ** 31 - 1).to(torch.int32)
    return x if x.is_contiguous() else x.contiguous()


def cached_positions(x, tokens: int, device, rotary: RotaryTable):
    """:func:`index_tensor` of positions of tokens that a cache counts as its
    own.  Device values are read back and checked like host values: the launch
    would leave a token outside the table out of its pages, which then show
    what they held before."""
    at = index_tensor(x, "positions", tokens, device, rotary.n_positions)
    if tokens and _torch().is_tensor(x) and x.device.type != "cpu":
        host = at.cpu().numpy()
        if host.min() < 0 or host.max() >= rotary.n_positions:
            raise ValueError(f"positions must lie in [0, {rotary.n_positions})")
    return at


def norm_rotate(queries, keys, positions, rotary: RotaryTable | None, *, q_weight=None, k_weight=None,
                eps: float = 1e-6, out=None):
    """``queries [T, Hq, hd]`` and ``keys [T, H, hd]`` (either may be None)
    normed per head with ``q_weight`` / ``k_weight`` (``[hd]`` or ``[heads,
    hd]``, any float type; None: no norm) and rotated to ``positions [T]``
    (int32 or int64 on the device, or host integers; ``rotary`` None: no
    rotation), in one launch.

    Returns ``(queries, keys)`` in the input's type, or writes ``out =
    (queries, keys)``: tensors of that type or fp32, which may be the inputs
    themselves but must not otherwise overlap them.  A device position outside
    the table gives NaN rows; a host one raises ValueError.
    """
    torch = _torch()
    first = queries if queries is not None else keys
    if first is None:
        raise ValueError("norm_rotate needs queries or keys")
    if first.dim() != 3:
        raise ValueError("queries and keys must have shape [tokens, heads, head_dim]")
    T, _, hd = first.shape
    device, dtype = first.device, first.dtype
    at, table = None, _NO_ROTARY
    if rotary is not None:
        if rotary.head_dim != hd:
            raise ValueError("the rotary table is for another head_dim")
        if rotary.table.device != device:
            raise ValueError(f"the rotary table must be on {device}")
        positions = index_tensor(positions, "positions", T, device, rotary.n_positions)
        at, table = positions.data_ptr(), rotary._c
    eps = float(eps)
    made, args = [], []
    for i, (x, w, name) in enumerate(((queries, q_weight, "queries"), (keys, k_weight, "keys"))):
        y = None if out is None else out[i]
        if x is None:
            args += _ABSENT
        else:
            if x.shape[0] != T or x.dtype != dtype:
                raise ValueError("queries and keys must have the same tokens and dtype")
            if out is None:
                y = torch.empty(x.shape, dtype=dtype, device=device)
            elif y is None or y.shape != x.shape or (y.dtype != dtype and y.dtype != torch.float32):
                raise ValueError(f"out must hold {name} of their shape, in their dtype or fp32")
            args += (token_rows(x, name, hd, device), head_norm(w, name + "' weight", x.shape[1], hd, eps, device),
                     token_rows(y, name + " out", hd, device))
        made.append(y)
    if T:
        call_on(device, _lib.lib().dc_norm_rotate, "dc_norm_rotate", T, hd, at, table, *args)
    return tuple(made)


__all__ = ["RotaryTable", "norm_rotate"]
