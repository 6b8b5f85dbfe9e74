"""Products with more rows or outputs than one launch holds blocks for."""
import pytest

from tests.test_gpu_projection import exact_case

pytestmark = pytest.mark.gpu


def test_rows_past_a_launch_of_their_preparation():
    """bf16 rows are prepared by a block each, 2^20 at most: 2^24 rows and a few, a
    block's later ones of other sizes than its first."""
    import torch

    from dotcache_amd.projection import project, workspace_bytes

    P, K, N, M = 4099, 128, 80, (1 << 24) + 77
    x, w, want, _ = exact_case(P, K, N, 32, True, "bf16")
    size = 2.0 ** (torch.arange(P, device="cuda") % 41 - 20)
    x, want = (x.double() * size[:, None]).bfloat16(), (want.double() * size[:, None]).bfloat16()
    assert workspace_bytes(w, x.dtype, M) >= M * K * 2  # (the tiles' kernel)
    many = x.repeat(-(-M // P), 1)[:M].contiguous()
    got = project(many, w)
    for r in range(0, M - M % P, P * 256):
        part = got[r: min(r + P * 256, M - M % P)].view(-1, P, N)
        assert bool((part == want).all())
    assert torch.equal(got[M - M % P:], want[: M % P])


def test_outputs_past_a_launch():
    """2^26 outputs and a few: the second portion has its own words, scales and columns."""
    import torch

    from dotcache_amd.projection import GroupedWeight, project

    P, K, N = 16 * 101, 8, (1 << 26) + 40
    x, w, want, _ = exact_case(2, K, P, 32, True, "f16")
    r = torch.Generator(device="cuda")
    r.manual_seed(3)
    codes = torch.randint(0, 16, (P, K), generator=r, device="cuda", dtype=torch.uint8)
    scales = (2.0 ** torch.randint(-1, 2, (P, 1), generator=r, device="cuda")).half()
    biases = (torch.randint(-16, 17, (P, 1), generator=r, device="cuda") / 2.0).half()
    want = (x.double() @ (codes.double() * scales.double() + biases.double()).t().contiguous()).half()
    at = torch.arange(N, device="cuda") % P
    w = GroupedWeight.from_codes(codes[at], scales[at], biases[at], group_size=32)
    got = project(x, w)
    for n in range(0, N, 1 << 22):
        assert torch.equal(got[:, n: n + (1 << 22)], want[:, at[n: n + (1 << 22)]])
