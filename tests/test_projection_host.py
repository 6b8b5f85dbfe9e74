"""4-bit weights' layout and refusals, on the CPU."""
import ctypes as C

import numpy as np
import pytest
import torch

from dotcache_amd import _lib
from dotcache_amd.projection import GroupedWeight, project


def make(N, K, gs, affine, seed=0, device="cpu"):
    """Codes, scales and biases [N, K], [N, G], and the matrix they stand for in fp64."""
    r = np.random.default_rng(seed)
    G = -(-K // gs)
    codes = r.integers(0, 16 if affine else 15, size=(N, K))
    scales = (r.random((N, G)) + 0.1).astype(np.float16)
    biases = (-8 * r.random((N, G))).astype(np.float16) if affine else None
    g = np.arange(K) // gs
    dense = codes * scales[:, g].astype(np.float64) + biases[:, g] if affine else (codes - 7) * scales[:, g].astype(np.float64)
    t = lambda x: None if x is None else torch.from_numpy(x).to(device)  # noqa: E731
    return t(codes.astype(np.uint8)), t(scales), t(biases), dense


@pytest.mark.parametrize("affine", [True, False])
@pytest.mark.parametrize("N,K,gs", [(1, 1, 32), (16, 128, 64), (17, 129, 128), (50, 300, 32), (33, 1000, 64)])
def test_layout(N, K, gs, affine):
    """Codes and scales lie where the header says, padding is 0, and dense() undoes it."""
    codes, scales, biases, dense = make(N, K, gs, affine)
    w = GroupedWeight.from_codes(codes, scales, biases, group_size=gs)
    at = C.c_int64()
    assert w.nbytes == _lib.lib().dc_grouped_weight_bytes(N, K, gs, int(affine), C.byref(at)) and w.shape == (N, K)
    data = w.data.numpy()
    nt, kt, ng = -(-N // 16), -(-K // 128), 128 // gs
    side = data[at.value:].view(np.float16).reshape(nt, kt, 16, ng, 2 if affine else 1)
    words = data[: at.value].view(np.uint32).reshape(nt * kt, 64, 4)
    for n in range(16 * nt):
        for k in range(0, 128 * kt, 1 if K < 400 else 37):
            lane, j = n % 16 + 16 * (k % 32 // 8), k % 8
            got = words[n // 16 * kt + k // 128, lane, k % 128 // 32] >> (4 * (j // 2 + 4 * (j % 2))) & 15
            assert got == (codes[n, k] if n < N and k < K else 0)
            s = side[n // 16, k // 128, n % 16, k % 128 // gs]
            inside = n < N and k // gs < scales.shape[1]
            assert s[0] == (scales[n, k // gs] if inside else 0) and (not affine or s[1] == (biases[n, k // gs] if inside else 0))
    assert np.array_equal(w.dense(torch.float64).numpy(), dense.astype(np.float32))
    for t in (torch.int8, torch.uint16, torch.int64):
        assert torch.equal(GroupedWeight.from_codes(codes.to(t), scales, biases, group_size=gs).data, w.data)


def test_weight_refusals():
    codes, scales, biases, _ = make(20, 100, 32, True)
    for c, s, b, gs in ((codes.float(), scales, biases, 32), (codes[0], scales, biases, 32), (codes, scales, biases, 48), (codes, scales.float(), biases, 32),
                        (codes, scales[:, :3], biases, 32), (codes, scales, biases[:5], 32), (codes + 1, scales, biases, 32),
                        (codes.to(torch.int16) - 1, scales, biases, 32), (torch.full_like(codes, 15), scales, None, 32),
                        (codes[:0], scales[:0], biases[:0], 32), (codes.bool(), scales, biases, 32), (codes, scales * float("nan"), biases, 32),
                        (codes, scales, biases * float("inf"), 32), (codes, torch.full_like(scales, 5000.0), biases, 32)):
        with pytest.raises(ValueError):
            GroupedWeight.from_codes(c, s, b, group_size=gs)
    for w, kw in ((torch.zeros(4, 64), {}), (torch.zeros(4, 64), dict(group_size=16)), (torch.zeros(64), {}), (torch.zeros(4, 0), {})):
        with pytest.raises(ValueError):
            GroupedWeight.quantize(w, **kw)


def test_call_refusals():
    codes, scales, biases, _ = make(20, 100, 32, True)
    w = GroupedWeight.from_codes(codes, scales, biases, group_size=32)
    x = torch.zeros(3, 100)
    for x, kw in ((torch.zeros(3, 99), {}), (torch.tensor(1.0), {}), (x.double(), {}), (torch.zeros(100, 3).t(), {}), (x, dict(out=torch.zeros(3, 19))),
                  (x, dict(out=torch.zeros(3, 20).half())), (x, dict(out=torch.zeros(20, 3).t())), (x, dict(out=torch.zeros(1, 20).expand(3, 20))),
                  (x[None], dict(out=torch.zeros(3, 20))), (x, {})):  # (the last: tensors on the CPU)
        with pytest.raises(ValueError):
            project(x, w, **kw)
    assert project(x[:0], w).shape == (0, 20)


def test_entry_refusals():
    L = _lib.lib()
    for a in ((0, 4, 32), (4, 0, 32), (4, 4, 16), (-1, 4, 32), (4, (1 << 30) + 1, 32), ((1 << 30) + 1, 4, 32)):
        assert L.dc_grouped_weight_bytes(*a, 1, None) == -1

    def call(rows=2, data=1 << 20, x=1 << 20, y=1 << 21, xd=0, yd=0, ys=20, gs=32):
        return L.dc_project(_lib.GroupedWeight(data, 20, 100, gs, 1), _lib.MatrixRows(x, 100, xd), _lib.MatrixRows(y, ys, yd), rows, None, 0, None)

    for kw in (dict(rows=-1), dict(data=0), dict(x=0), dict(y=0), dict(xd=3), dict(yd=1), dict(ys=19), dict(gs=48), dict(data=(1 << 20) + 8),
               dict(x=(1 << 20) + 2), dict(y=(1 << 20) + 1, xd=1, yd=1)):
        assert call(**kw) == _lib.DC_EINVAL, kw
    assert call(rows=0) == _lib.DC_OK
