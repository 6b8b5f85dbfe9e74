"""Weights of the products one by one: rows with a single 1 bring out single
weights, in calls that the tiles' kernel takes."""
import numpy as np
import pytest

from tests.test_gpu_chunk import _dt

pytestmark = pytest.mark.gpu


def _levels(N, K, gs, affine, seed):
    """Codes, fp16 scales and biases of many sizes and either sign, some
    groups with a level that is exactly 0, and the levels in fp64 (exact)."""
    import torch

    r = np.random.default_rng(seed)
    G = -(-K // gs)
    codes = r.integers(0, 16 if affine else 15, size=(N, K))
    scales = (r.choice([-1.0, 1.0], size=(N, G)) * 2.0 ** r.uniform(-9, 6, size=(N, G))).astype(np.float16)
    biases = None
    if affine:
        biases = (scales.astype(np.float64) * -r.uniform(-4, 20, size=(N, G))).astype(np.float16)
        zero = r.random((N, G)) < 0.5  # 2 s and 4 s are fp16 values: codes 2 and 4 stand for 0
        biases = np.where(zero, -scales * r.choice(np.array([2, 4], dtype=np.float16), size=(N, G)), biases).astype(np.float16)
        scales[0, 0], biases[0, 0], codes[0, 0] = 1.0732421875, -2.146484375, 2
    g = np.arange(K) // gs
    s = scales.astype(np.float64)[:, g]
    dense = codes * s + biases.astype(np.float64)[:, g] if affine else (codes - 7) * s
    put = lambda x: None if x is None else torch.from_numpy(x).cuda()  # noqa: E731
    return put(codes.astype(np.uint8)), put(scales), put(biases), dense


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("gs,affine", [(32, True), (64, True), (128, True), (32, False), (64, False), (128, False)])
def test_single_weights_of_large_calls(gs, affine, dtype):
    """An output is its weight rounded to fp16 once (products with 1 and 0 and
    their sums are exact), then to the rows' type."""
    import torch

    from dotcache_amd.projection import GroupedWeight, project, workspace_bytes

    M, K, N = 1152, 320, 1100
    codes, scales, biases, dense = _levels(N, K, gs, affine, gs)
    w = GroupedWeight.from_codes(codes, scales, biases, group_size=gs)
    assert workspace_bytes(w, torch.bfloat16, M) > 0  # (a call of the tiles' kernel)
    x = torch.zeros(M, K, device="cuda", dtype=_dt(dtype))
    at = np.arange(M) % K
    x[torch.arange(M, device="cuda"), torch.from_numpy(at).cuda()] = 1.0
    got = project(x, w)
    want = torch.from_numpy(dense.astype(np.float16)).cuda().t()[torch.from_numpy(at).cuda()].to(_dt(dtype))
    assert torch.equal(got, want), float((got.double() - want.double()).abs().max())
    if affine:
        assert bool((want == 0).any())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M", [5, 16, 40, 200])
def test_single_weights_of_small_calls(M, dtype):
    """Those of the other kernels are not rounded: an output is s sum x (16 + c)
    + (b - 16 s) sum x in fp32 (2^-24 of each of the two terms and of the
    offset), then rounded to the rows' type."""
    import torch

    from dotcache_amd.projection import GroupedWeight, project, workspace_bytes

    K, N, gs = 320, 70, 32
    half = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
    for affine in (True, False):
        codes, scales, biases, dense = _levels(N, K, gs, affine, M)
        w = GroupedWeight.from_codes(codes, scales, biases, group_size=gs)
        assert workspace_bytes(w, torch.bfloat16, M) == 0
        x = torch.zeros(M, K, device="cuda", dtype=_dt(dtype))
        at = np.arange(M) * 7 % K
        x[torch.arange(M, device="cuda"), torch.from_numpy(at).cuda()] = 1.0
        got, want = project(x, w).double().cpu().numpy(), dense.T[at]
        g = at // gs
        s = scales.double().cpu().numpy().T[g]
        off = biases.double().cpu().numpy().T[g] - 16 * s if affine else -23 * s
        bound = 2.0 ** -24 * (31 * np.abs(s) + 2 * np.abs(off) + np.abs(want)) + half * np.abs(want) + 2.0 ** -25 * (dtype == "f16")
        assert np.all(np.abs(got - want) <= bound * (1 + 2.0 ** -10)), float(np.max(np.abs(got - want) / bound))


@pytest.mark.parametrize("M", [3, 40, 1152])
def test_levels_at_the_ends_of_fp16(M):
    """Levels within fp16's range, of scales that 15 times leave it."""
    import torch

    from dotcache_amd.projection import GroupedWeight, project

    K, N, gs = 128, 1100, 32
    r = np.random.default_rng(M)
    codes = r.integers(0, 16, size=(N, K))
    flip = r.choice([-1.0, 1.0], size=(N, 4))
    scales, biases = (flip * r.uniform(8000, 8700, size=(N, 4))).astype(np.float16), (flip * -65504.0).astype(np.float16)
    g = np.arange(K) // gs
    dense = codes * scales.astype(np.float64)[:, g] + biases.astype(np.float64)[:, g]
    assert np.all(np.abs(dense) <= 65504) and np.any(np.abs(15 * scales.astype(np.float64)) > 65504)
    w = GroupedWeight.from_codes(*(torch.from_numpy(x).cuda() for x in (codes.astype(np.uint8), scales, biases)), group_size=gs)
    x = torch.zeros(M, K, device="cuda", dtype=torch.float16)
    at = np.arange(M) % K
    x[torch.arange(M, device="cuda"), torch.from_numpy(at).cuda()] = 0.5
    got = project(x, w).double().cpu().numpy()
    want = 0.5 * dense.T[at]
    # fp16's rounding of a weight (many rows) and of the output, half a step each; sums of 31 scale in fp32 (a few rows)
    assert np.all(np.abs(got - want) <= 2.0 ** -10 * np.abs(want) + 8700 * 40 * 2.0 ** -23)
