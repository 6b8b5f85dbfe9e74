"""The products' kernels for 17 rows up, each at sizes that its rule sends to
it: bounds without an allowance that another kernel needs."""
import numpy as np
import pytest

from tests.test_gpu_chunk import _dt
from tests.test_gpu_projection import HALF, exact_case
from tests.test_projection_host import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("M", [17, 33, 64, 200])
def test_rows_of_exact_weights(M, dtype):
    """17 rows to a few hundred at 100 outputs: codes and rows are exact operands, so
    an output is off by its sums' fp32 roundings (2^-23 for each of a group's terms and of the
    groups, of at most (31 scale + |offset|) |x|) and by its own alone."""
    import torch

    from dotcache_amd.projection import GroupedWeight, project, workspace_bytes

    K, N, gs = 700, 100, 64
    codes, scales, biases, dense = make(N, K, gs, True, M, "cuda")
    w = GroupedWeight.from_codes(codes, scales, biases, group_size=gs)
    assert workspace_bytes(w, torch.bfloat16, M) == 0  # (not the tiles' kernel)
    r = np.random.default_rng(M)
    x = torch.from_numpy((r.normal(size=(M, K)) * np.exp(r.normal(size=(1, K)))).astype(np.float32)).to(_dt(dtype)).cuda()
    got, xs = project(x, w).double().cpu().numpy(), x.double().cpu().numpy()
    want = xs @ dense.T
    g = np.arange(K) // gs
    s, b = (t.double().cpu().numpy()[:, g] for t in (scales, biases))
    size = np.abs(xs) @ (31 * s + np.abs(b - 16 * s)).T
    bound = (gs + -(-K // gs) + 16) * 2.0 ** -23 * size + HALF[dtype] * np.abs(want)
    assert np.all(np.abs(got - want) <= bound), float(np.max(np.abs(got - want) / bound))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("M,K,N", [(1100, 300, 1100), (1152, 320, 2688)])
def test_tiles_keep_values_that_are_not_finite_in_their_rows(M, K, N, dtype):
    import torch

    from dotcache_amd.projection import project, workspace_bytes

    x, w, want, _ = exact_case(M, K, N, 64, True, dtype)
    assert workspace_bytes(w, torch.bfloat16, M) > 0
    bad = [1, 95, 96, M - 1]
    for i, v in zip(bad, (float("inf"), float("nan"), -float("inf"), float("nan"))):
        x[i, (37 * i) % K] = v
    got = project(x, w)
    rows = [i for i in range(M) if i not in bad]
    assert torch.equal(got[rows], want[rows]) and not torch.isfinite(got[bad]).any()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_tiles_over_the_range_of_their_type(dtype):
    """Rows scaled by powers of two from end to end of their type; within a bf16 row, values
    2^60 apart: the small ones count to 2^-39 of the largest, as fp32 sums would lose them too."""
    import torch

    from dotcache_amd.projection import project, workspace_bytes

    M, K, N = 1100, 160, 1100
    x, w, _, dense = exact_case(M, K, N, 32, True, dtype)
    assert workspace_bytes(w, torch.bfloat16, M) > 0
    d = dense.t().contiguous()
    for f in ((2.0 ** 5, 2.0 ** -10) if dtype == "f16" else (2.0 ** 100, 2.0 ** -100, 2.0 ** -125)):
        y = x * f
        assert torch.equal(project(y, w), (y.double() @ d).to(y.dtype)), f
    if dtype == "bf16":
        y = x.clone()
        y[:, :32] *= 2.0 ** 60
        got, want = project(y, w).double(), y.double() @ d
        top = y.double().abs().amax(1, keepdim=True)
        lost = (2.0 ** -39 * top) * d.abs().sum(0)[None] + (K + 8) * 2.0 ** -23 * (y.double().abs() @ d.abs())
        assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + lost).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_calls_repeat_their_bits(dtype):
    """Sums are joined in a fixed order."""
    import torch

    from dotcache_amd.projection import GroupedWeight, project

    codes, scales, biases, _ = make(1100, 1000, 32, True, 1, "cuda")
    w = GroupedWeight.from_codes(codes, scales, biases, group_size=32)
    r = torch.Generator(device="cuda")
    r.manual_seed(1)
    for M in (1, 16, 40, 200, 1100):
        x = torch.randn(M, 1000, generator=r, device="cuda").to(_dt(dtype))
        first = project(x, w)
        for _ in range(4):
            assert torch.equal(project(x, w), first), M


def test_two_streams_at_once():
    """Calls that overlap have workspaces of their own."""
    import torch

    from dotcache_amd.projection import project

    cases = [exact_case(M, K, 1100, 64, True, "bf16", M) for M, K in ((1100, 300), (1152, 320), (40, 384))]
    streams = [torch.cuda.Stream() for _ in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[] for _ in cases]
    for _ in range(8):
        for (x, w, _, _), s, out in zip(cases, streams, got):
            with torch.cuda.stream(s):
                out.append(project(x, w))
    torch.cuda.synchronize()
    for (_, _, want, _), out in zip(cases, got):
        assert all(torch.equal(y, want) for y in out)
