"""Gaps that are not their items' own: the kernels leave them out of account."""
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
