"""Gaps that are not their items' own: the kernels leave them out of account.
Ranges of a token that overlap: what both hold counts once."""
import dataclasses

import numpy as np
import pytest

from dotcache_amd.chunk import ChunkMask
from tests.test_gpu_chunk import _Batch
from tests.test_gpu_chunk_rule import check_rule

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new", [[9, 2], [300, 40]])
def test_gaps_outside_their_items(new, dtype):
    """Empty ones, reversed ones, ones that reach past the item on either side:
    the ranges alone say what a row attends, so outputs stay right."""
    import torch

    rng = np.random.default_rng(sum(new))
    batch = _Batch(rng, [1900, 1500], 2, 64, 64, "a4", "s4")
    mask = ChunkMask(window=129, sinks=4)
    plan = batch.plan(new, 4, mask=mask, target_items=1)
    g = plan.host_gaps
    assert bool((g[:, 0] > 0).any())
    begin, end = plan.host_items[:, 6], plan.host_items[:, 7]
    for name, bad in (("empty", np.stack([g[:, 0], g[:, 0]], 1)), ("reversed", g[:, ::-1]), ("ahead", np.stack([begin, g[:, 1]], 1)),
                      ("behind", np.stack([g[:, 0], end], 1)), ("far", np.stack([g[:, 0], np.full(len(g), 2 ** 31 - 1)], 1)),
                      ("before", np.stack([begin - 128, begin - 64], 1))):
        print(f"chunk gaps {new} {dtype} {name}", flush=True)
        other = dataclasses.replace(plan, gaps=torch.from_numpy(np.ascontiguousarray(bad, dtype=np.int32)).cuda())
        check_rule(batch, new, 4, dtype, rng, mask=mask, cap=5.0, plan=other)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("new", [[150, 30, 1], [3, 2, 1]])
def test_ranges_that_overlap(new, dtype):
    rng = np.random.default_rng(len(dtype) + new[0])
    batch = _Batch(rng, [700, 30, 250], 2, 128, 64, "a4", "a4")
    r, t = np.zeros((sum(new), 4), dtype=np.int64), 0
    for n, c in zip(new, batch.ctx):
        r[t: t + n] = np.concatenate([np.sort(rng.integers(0, c + 1, size=(n, 2)), axis=1) for _ in range(2)], axis=1)
        t += n
    r[0] = [0, 700, 0, 700]  # twice the same
    r[1] = [100, 600, 200, 300]  # one inside the other
    for cap, slopes in ((None, True), (4.0, False)):
        print(f"chunk overlaps {new} {dtype} {cap}", flush=True)
        check_rule(batch, new, 3, dtype, rng, mask=r, cap=cap, slopes=slopes, validate=True)
