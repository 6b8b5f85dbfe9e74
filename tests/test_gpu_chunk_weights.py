"""Chunk attention where one token outweighs thousands of others that together
still count: weights far below a row's largest are not lost in fp16."""
import numpy as np
import pytest

from tests.test_gpu_chunk import _Batch, _dt, _want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("value", ["m3", "m3_f32"])
@pytest.mark.parametrize("n,n_q", [(2, 2), (5, 7), (80, 2)])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_many_small_weights(hd, n, n_q, value, dtype):
    """The first key gives a logit of 18 and a value of 0, every other a logit
    of 0 and a value of 1: e^-18 (2^-26) each, 6e-5 in all.

    A weight is held against 2^7 at least for the largest, so its rounding in
    fp16 (2^-11 relative, in steps of 2^-24 at the least: 2^-25 off) is off by
    2^-32 of the largest at most; beside it the logits (exact here but for
    2^-20), the sums and the output's own rounding (half its smallest step)."""
    import torch

    rng = np.random.default_rng(hd)
    ctx, P = 4096, 64
    print(f"chunk small weights {hd} {n}x{n_q} {value} {dtype}", flush=True)
    batch = _Batch(rng, [ctx], 1, hd, P, "m3", value, tail=False)
    rows = [np.zeros((ctx, hd), np.float32), np.ones((ctx, hd), np.float32)]
    rows[0][0, 0], rows[1][0] = 18.0, 0.0
    t = np.arange(ctx)
    for pool, table, x in zip(batch.pools, batch.host, rows):
        pool.encode_rows(torch.from_numpy(x).cuda(), table[0, 0, t // P], (t % P).astype(np.int32))
    batch.read()
    assert np.array_equal(batch.rows[0][0, 0], rows[0]) and np.array_equal(batch.rows[1][0, 0], rows[1])
    q = torch.zeros(n, n_q, hd, device="cuda", dtype=_dt(dtype))
    q[..., 0] = 1.0
    want, size, _ = _want(batch, q.double().cpu().numpy(), [n], n_q, 1.0)
    assert np.all((want > 5e-5) & (want < 7e-5))
    got = batch.attend(q, batch.plan([n], n_q, dtype=q.dtype, target_items=1), 1.0).double().cpu().numpy()
    half = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
    weights = ctx * 2.0 ** -24 * size if dtype == "f32" else ctx * 2.0 ** -32 + ctx * 2.0 ** -24 * size
    bound = weights + (half + 2.0 ** -10) * want + (2.0 ** -25 if dtype == "f16" else 0)
    assert np.all(np.abs(got - want) <= bound), float(np.max(np.abs(got - want) / bound))
