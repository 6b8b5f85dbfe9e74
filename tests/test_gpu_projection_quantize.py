"""Dense matrices that no levels stand for are refused."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("scheme", ["affine", "symmetric"])
def test_quantize_refuses_what_is_not_finite(scheme, bad):
    import torch

    from dotcache_amd.projection import GroupedWeight

    for at in ((0, 0), (39, 99)):
        for dtype in (torch.float32, torch.bfloat16):
            w = torch.randn(40, 100, device="cuda").to(dtype)
            w[at] = bad
            with pytest.raises(ValueError):
                GroupedWeight.quantize(w, group_size=32, scheme=scheme)
