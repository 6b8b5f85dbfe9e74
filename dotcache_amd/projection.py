"""Rows times weight matrices held in 4 bits (``dc_project``): the products that
make a layer's queries, keys and values ahead of the cache, and those behind its
attention.

A weight ``W [outputs, inputs]`` has 4-bit codes with an fp16 scale, and with the
affine scheme an fp16 bias, for every group of 32, 64 or 128 inputs of an output,
the levels of the caches' pages:

    W = scale * code + bias          (affine, codes 0 .. 15)
    W = scale * (code - 7)           (symmetric, codes 0 .. 14)

Codes, rows and their products are exact as matrix operands and sums are fp32,
so an output is rounded once, to the rows' type.  Calls of many 16-bit rows, bound by
the matrix instructions and not by the weights' bytes, round each weight to fp16
besides (once, 2^-11): those of more than 64 rows for which the tiles' kernel, by rows
and outputs, is done first.  So fp16 rows among hundreds are less precise than
alone: off by 2.8e-4 of their size instead of the output's own rounding, 2.1e-4 (bf16
1.67e-3 instead of 1.66e-3).  For inference: no gradient flows through a
product.  The reference leaves these
products to its models (reference ``dotcache/integrations/llama.py:345-358``,
``:476-481``); its levels are those of ``dotcache/modes/m0_affine.py:15-90``.
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from .page_pool import call_on, dtype_code

GROUP_SIZES = (32, 64, 128)
_TILE_N, _TILE_K = 16, 128
_QUANTIZE_ROWS = 256  # groups to a page while a matrix is encoded


def _torch():
    import torch

    return torch


class GroupedWeight:
    """A weight matrix of 4-bit codes on the device, in the order in which the
    kernels read it (``dc_grouped_weight``).  :meth:`quantize` makes it from a
    dense matrix, :meth:`from_codes` from a checkpoint's codes, and the class
    itself from the ``data`` of another (a saved one's, or moved to another device)."""

    def __init__(self, data, outputs: int, inputs: int, group_size: int, affine: bool):
        outputs, inputs, gs = int(outputs), int(inputs), _group_size(group_size)
        need = int(_lib.lib().dc_grouped_weight_bytes(outputs, inputs, gs, int(bool(affine)), None))
        if need < 0:
            raise ValueError("a weight needs outputs and inputs, 2^30 of each at most")
        if data.dtype != _torch().uint8 or data.dim() != 1 or data.numel() != need or not data.is_contiguous() or data.data_ptr() % 16:
            raise ValueError(f"a weight's data must be {need} contiguous bytes, 16-byte aligned")
        self._data, self.outputs, self.inputs = data, outputs, inputs
        self.group_size, self.affine = gs, bool(affine)
        self._c = _lib.GroupedWeight(data.data_ptr(), outputs, inputs, gs, int(self.affine))

    @property
    def data(self):
        """uint8, the bytes of ``dc_grouped_weight`` (read only: the calls keep its address)."""
        return self._data

    @property
    def shape(self) -> tuple[int, int]:
        return self.outputs, self.inputs

    @property
    def device(self):
        return self.data.device

    @property
    def nbytes(self) -> int:
        return self.data.numel()

    @classmethod
    def from_codes(cls, codes, scales, biases=None, *, group_size: int) -> "GroupedWeight":
        """``codes [outputs, inputs]`` (any integer type, 0 .. 15), ``scales`` and
        ``biases`` (None: symmetric, codes 0 .. 14) ``[outputs, ceil(inputs /
        group_size)]`` fp16, all on one device."""
        torch = _torch()
        gs = _group_size(group_size)
        if codes.dim() != 2 or codes.dtype.is_floating_point or codes.dtype.is_complex or codes.dtype == torch.bool:
            raise ValueError("codes must be integers of shape [outputs, inputs]")
        N, K = codes.shape
        if N == 0 or K == 0:
            raise ValueError("a weight needs outputs and inputs")
        G = -(-K // gs)
        for x, name in ((scales, "scales"), (biases, "biases")):
            if x is None and name == "biases":
                continue
            if tuple(x.shape) != (N, G) or x.dtype != torch.float16 or x.device != codes.device:
                raise ValueError(f"{name} must be fp16 [{N}, {G}] on the codes' device")
        _check_levels(scales, biases)
        most = 15 if biases is not None else 14
        data = _new_data(N, K, gs, biases is not None, codes.device)
        # rows in portions: a portion's codes are widened (to 64 bits for their check, so that none wraps into the range)
        step = max(_TILE_N, (1 << 24) // K // _TILE_N * _TILE_N)
        for r in range(0, N, step):
            part = codes[r: r + step].to(torch.int64)
            if int(part.min()) < 0 or int(part.max()) > most:
                raise ValueError(f"codes must lie in [0, {most}]")
            part = torch.nn.functional.pad(part.to(torch.int32), (0, -K % _TILE_K, 0, -part.shape[0] % _TILE_N))
            _put(data, N, K, gs, r, part.unflatten(-1, (-1, 8)), scales[r: r + step], None if biases is None else biases[r: r + step])
        return cls(data, N, K, gs, biases is not None)

    @classmethod
    def quantize(cls, weight, *, group_size: int = 64, scheme: str = "affine") -> "GroupedWeight":
        """``weight [outputs, inputs]`` (fp32, fp16 or bf16, on the device) to
        the levels that the page encoder gives its groups."""
        torch = _torch()
        from .page_pool import DevicePagePool, PoolGeometry, page_format_of

        gs = _group_size(group_size)
        if weight.dim() != 2 or weight.shape[0] == 0 or weight.shape[1] == 0:
            raise ValueError("weight must have shape [outputs, inputs]")
        dtype_code(weight)
        if weight.device.type != "cuda":
            raise ValueError("quantize: the weight must be on a GPU")
        N, K = weight.shape
        fmt = page_format_of("M0", scheme, 4)
        affine, G, P = scheme == "affine", -(-K // gs), _QUANTIZE_ROWS
        data = _new_data(N, K, gs, affine, weight.device)
        step = max(_TILE_N, (1 << 24) // K // _TILE_N * _TILE_N)
        with torch.cuda.device(weight.device):
            for r in range(0, N, step):
                # every group as a row of its own, one page after another
                part = weight[r: r + step]
                if not bool(torch.isfinite(part).all()):
                    raise ValueError("quantize: the weight must be finite")
                rows = torch.nn.functional.pad(part, (0, -K % gs)).reshape(-1, gs)
                n, pages = rows.shape[0], -(-rows.shape[0] // P)
                pool = DevicePagePool(PoolGeometry(gs, gs, P), device=weight.device, reserve_pages=pages,
                                      reserve_bytes=pages * _lib.page_blob_bytes(*fmt, _lib.geometry(gs, gs, P)))
                ids = pool.allocate(*fmt, pages, tokens=P)
                at = torch.arange(n, device=weight.device, dtype=torch.int32)
                pool.encode_rows(rows, torch.from_numpy(ids).to(weight.device)[(at // P).long()], at % P)
                blobs = pool.arena[: pages * pool.blob_bytes(*fmt)].view(pages, -1)
                codes = blobs[:, : P * gs // 2].reshape(pages * P, gs // 2)[:n]
                codes = torch.stack([codes & 15, codes >> 4], dim=-1).reshape(-1, G * gs).to(torch.int32)
                side = [blobs[:, o: o + 2 * P].contiguous().view(torch.float16).reshape(-1)[:n].view(-1, G)
                        for o in range(P * gs // 2, P * gs // 2 + (4 if affine else 2) * P, 2 * P)]
                codes[:, K:] = 0
                _check_levels(side[0], side[1] if affine else None)
                codes = torch.nn.functional.pad(codes, (0, -K % _TILE_K - (G * gs - K), 0, -codes.shape[0] % _TILE_N))
                _put(data, N, K, gs, r, codes.unflatten(-1, (-1, 8)), side[0], side[1] if affine else None)
        return cls(data, N, K, gs, affine)

    def dense(self, dtype=None):
        """The matrix ``[outputs, inputs]`` that codes, scales and biases stand
        for (fp32, or ``dtype``: rounded once)."""
        torch = _torch()
        N, K, gs = self.outputs, self.inputs, self.group_size
        words, side = _views(self.data, N, K, gs, self.affine)
        shift = torch.arange(8, device=self.device, dtype=torch.int32)
        shift = 4 * (shift // 2 + 4 * (shift % 2))
        # [nt, kt, g, row, w, j] -> [nt, row, kt, w, g, j]
        codes = ((words[..., None] >> shift) & 15).permute(0, 3, 1, 4, 2, 5).reshape(words.shape[0] * _TILE_N, -1, gs)
        side = side.permute(0, 2, 1, 3, 4).reshape(codes.shape[0], codes.shape[1], -1).float()
        x = side[..., :1] * codes + side[..., 1:] if self.affine else side * (codes - 7)
        return x.reshape(codes.shape[0], -1)[:N, :K].to(dtype or torch.float32)


def _group_size(group_size) -> int:
    if group_size not in GROUP_SIZES:
        raise ValueError("group_size must be 32, 64 or 128")
    return int(group_size)


def _check_levels(scales, biases) -> None:
    """Every level is one that fp16 holds (those between lie within the outer two)."""
    s = scales.float()
    top = (s * 7).abs() if biases is None else _torch().maximum(biases.float().abs(), (s * 15 + biases.float()).abs())
    if not float(top.max()) <= 65504.0:
        raise ValueError("a weight's scales, biases and levels must lie in fp16's range")


def _new_data(N: int, K: int, gs: int, affine: bool, device):
    n = int(_lib.lib().dc_grouped_weight_bytes(N, K, gs, int(affine), None))
    return _torch().zeros(n, dtype=_torch().uint8, device=device)


def _views(data, N: int, K: int, gs: int, affine: bool):
    """The codes' words ``[N tiles, K tiles, 4, 16, 4]`` and the scales ``[N
    tiles, K tiles, 16, groups, 1 or 2]`` in a weight's bytes."""
    torch = _torch()
    nt, kt = -(-N // _TILE_N), -(-K // _TILE_K)
    words = data[: nt * kt * 1024].view(torch.int32).view(nt, kt, 4, _TILE_N, 4)
    return words, data[nt * kt * 1024:].view(torch.float16).view(nt, kt, _TILE_N, _TILE_K // gs, 2 if affine else 1)


def _put(data, N: int, K: int, gs: int, first: int, codes, scales, biases) -> None:
    """Rows from ``first`` (a multiple of 16) on: ``codes [rows, inputs / 8, 8]``,
    padded to whole tiles, and their groups' scales and biases."""
    torch = _torch()
    words, side = _views(data, N, K, gs, biases is not None)
    rows, kt = codes.shape[0], -(-K // _TILE_K)
    at = slice(first // _TILE_N, (first + rows) // _TILE_N)
    w = torch.zeros(codes.shape[:2], dtype=torch.int32, device=codes.device)
    for j in range(8):
        w |= codes[..., j] << (4 * (j // 2 + 4 * (j % 2)))
    # [nt, row, kt, w, g] -> [nt, kt, g, row, w]
    words[at] = w.view(-1, _TILE_N, kt, 4, 4).permute(0, 2, 4, 1, 3)
    pad = (0, kt * (_TILE_K // gs) - scales.shape[1], 0, rows - scales.shape[0])
    for i, x in enumerate((scales, biases)):
        if x is not None:
            side[at, :, :, :, i] = torch.nn.functional.pad(x, pad).view(-1, _TILE_N, kt, _TILE_K // gs).transpose(1, 2)


def workspace_bytes(weight: GroupedWeight, dtype, rows: int) -> int:
    """Bytes of :func:`project`'s workspace for ``rows`` rows of ``dtype``."""
    return int(_lib.lib().dc_project_workspace_bytes(weight._c, dtype_code(_torch().empty(0, dtype=dtype)), int(rows)))


def project(x, weight: GroupedWeight, *, out=None, workspace=None):
    """``x [..., inputs]`` (fp32, fp16 or bf16; rows at any stride, their
    elements contiguous) times the weight's transpose: ``[..., outputs]`` in the
    same type.  ``out`` (two-dimensional like ``x``, rows at any stride that does
    not overlap) receives it instead; it must not overlap ``x``.  An infinity or
    NaN in a row makes that row's outputs infinities or NaN; so may finite values
    so large that 31 times their sum over a group, or that times the scale, leaves
    fp32 (from 2^115 on, at scales up to 1).  ``workspace``: uint8,
    :func:`workspace_bytes` at least, 16-byte aligned, not shared by calls that may
    overlap (default: one of its own where a call needs it)."""
    shape = x.shape
    if not shape or shape[-1] != weight.inputs:
        raise ValueError(f"rows must have shape [..., {weight.inputs}]")
    if x.device != weight.device:
        raise ValueError(f"rows must be on {weight.device}")
    code = dtype_code(x)
    rows = x if len(shape) == 2 else x.reshape(-1, weight.inputs)
    stride = rows.stride()
    if stride[1] != 1 and weight.inputs > 1:
        raise ValueError("rows must have contiguous elements")
    if out is None:
        y = x.new_empty((rows.shape[0], weight.outputs))  # (1 us of the host's time less than torch.empty)
    else:
        y = out
        if len(shape) != 2 or tuple(y.shape) != (rows.shape[0], weight.outputs) or y.dtype != x.dtype or y.device != x.device:
            raise ValueError(f"out must have shape [{rows.shape[0]}, {weight.outputs}], the rows' dtype and device")
        if weight.outputs > 1 and y.stride(1) != 1 or y.shape[0] > 1 and y.stride(0) < weight.outputs:
            raise ValueError("out must have contiguous elements, and rows that do not overlap")
    n = rows.shape[0]
    if n:
        L = _lib.lib()
        need = L.dc_project_workspace_bytes(weight._c, code, n) if n > 64 else 0
        if need == 0:
            workspace = None
        elif workspace is None:
            workspace = x.new_empty(need, dtype=_torch().uint8)
        elif workspace.numel() * workspace.element_size() < need or not workspace.is_contiguous() or workspace.device != x.device:
            raise ValueError(f"workspace must be contiguous, {need} bytes at least, on {x.device}")
        elif workspace.data_ptr() % 16:
            raise ValueError("workspace must be 16-byte aligned")
        call_on(x.device, L.dc_project, "dc_project", weight._c, _lib.MatrixRows(rows.data_ptr(), stride[0], code),
                _lib.MatrixRows(y.data_ptr(), y.stride(0), code), n, None if workspace is None else workspace.data_ptr(), need)
    return y if len(shape) == 2 else y.view(*shape[:-1], weight.outputs)


__all__ = ["GroupedWeight", "project", "workspace_bytes"]
