"""Chunk attention under scales that are not positive and weights far below a
row's largest, against fp64 numpy on the pages' own values, for each kernel:
few rows and row tiles of 16-bit queries, the general kernel in both types."""
import numpy as np
import pytest

from tests.test_gpu_chunk import _Batch, _bound, _dt, _want

pytestmark = pytest.mark.gpu

# (key, value, new tokens of two sequences, queries): few rows; row tiles; formats
# that the general kernel takes; fp32 queries
_KERNELS = [("a4", "s4", [5, 3], "f16"), ("m3", "s8", [5, 3], "bf16"), ("a4", "s4", [90, 70], "f16"), ("s8", "m3", [90, 70], "bf16"),
            ("s2", "a3", [60, 5], "f16"), ("m3_f32", "a2", [9, 31], "bf16"), ("a4", "s4", [40, 5], "f32")]


@pytest.mark.parametrize("key,value,new,dtype", _KERNELS)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_scales_that_are_not_positive(hd, key, value, new, dtype):
    """A negative scale is the positive one of the negated queries, a scale of 0
    the mean of the values that a row sees; tokens that it does not see, in
    tiles that some rows see in part and behind the last token, stay out."""
    import torch

    rng = np.random.default_rng(hd + len(new))
    print(f"chunk scale {hd} {key} {value} {new} {dtype}", flush=True)
    batch = _Batch(rng, [150, 331], 2, hd, 32, key, value)
    n_q, scale = 3, 1.0 / np.sqrt(hd)
    q = torch.from_numpy((0.5 * rng.normal(size=(sum(new), 2 * n_q, hd))).astype(np.float32)).to(_dt(dtype)).cuda()
    q64, vmax = q.double().cpu().numpy(), np.max(np.abs(batch.rows[1]))
    for target in (None, 1):  # (ranges cut, and whole)
        plan = batch.plan(new, n_q, dtype=q.dtype, **({} if target is None else dict(target_items=target)))
        down = batch.attend(q, plan, -scale)
        assert torch.equal(down, batch.attend(-q, plan, scale))
        flat = batch.attend(q, plan, 0.0)
        for got, rows, s in ((down, -q64, scale), (flat, 0 * q64, 1.0)):
            want, size, logit = _want(batch, rows, new, n_q, s)
            bound = _bound(dtype, want, size, logit, max(batch.ctx), hd, vmax)
            err = np.abs(got.double().cpu().numpy() - want)
            assert np.all(err <= bound), float(np.max(err / bound))
