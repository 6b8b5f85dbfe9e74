"""Chunk attention of 16-bit queries at every width, by the rows of a call and
the page size: each size of the few-row kernel (to 16, 32 and 48 rows) and the
row tiles, over pages that tiles fit, pages that only some wavefronts' tokens
fit and pages that none do."""
import numpy as np
import pytest

from tests.test_gpu_chunk import _Batch, _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [3, 5, 7, 20])  # query heads of the five new tokens: 15, 25, 35 and 100 rows
@pytest.mark.parametrize("P", [10, 16, 48, 64])
@pytest.mark.parametrize("hd", [64, 96, 128, 256])
def test_rows_and_pages(hd, P, rows, dtype):
    for seed, (key, value) in enumerate([("m3", "s4"), ("a4", "m3"), ("s8", "a8")]):
        rng = np.random.default_rng(1000 * hd + 10 * P + seed)
        print(f"chunk instance {hd} pages of {P} {5 * rows} rows {key} {value} {dtype}", flush=True)
        batch = _Batch(rng, [203, 64], 1, hd, P, key, value)
        _check(batch, [5, 5], rows, dtype, rng)


@pytest.mark.parametrize("P", [16, 64])
@pytest.mark.parametrize("hd,n_q", [(64, 9), (128, 7), (96, 5), (256, 3)])
def test_one_long_range_of_few_rows(hd, n_q, P):
    """Drafted tokens behind a range that is cut, and one of many tiles."""
    rng = np.random.default_rng(hd + P)
    print(f"chunk few rows {hd} x {n_q} pages of {P}", flush=True)
    batch = _Batch(rng, [1500], 1, hd, P, "a4", "s4")
    for target in (1, 64):
        _check(batch, [5], n_q, "bf16", rng, plan=batch.plan([5], n_q, target_items=target))
