"""A 4-bit weight made of another's bytes, on the CPU."""
import pytest
import torch

from dotcache_amd.projection import GroupedWeight
from tests.test_projection_host import make


def _weight(N=20, K=200, gs=64):
    codes, scales, biases, _ = make(N, K, gs, True)
    return GroupedWeight.from_codes(codes, scales, biases, group_size=gs)


def test_the_same_bytes_are_the_same_weight():
    w = _weight()
    again = GroupedWeight(w.data.clone(), 20, 200, 64, True)
    assert torch.equal(again.dense(), w.dense()) and again.shape == (20, 200) and again.nbytes == w.nbytes


@pytest.mark.parametrize("change", [
    lambda d: (d[:-1], 20, 200, 64, True), lambda d: (d[:0], 20, 200, 64, True), lambda d: (d, 33, 200, 64, True),
    lambda d: (d, 20, 257, 64, True), lambda d: (d, 20, 200, 32, True), lambda d: (d, 20, 200, 64, False), lambda d: (d, 20, 200, 48, True),
    lambda d: (d, 0, 200, 64, True), lambda d: (d, 20, -1, 64, True), lambda d: (d.view(torch.int8), 20, 200, 64, True),
    lambda d: (d.view(-1, 2), 20, 200, 64, True), lambda d: (torch.cat([d, d])[::2], 20, 200, 64, True),
    lambda d: (torch.cat([d[:8], d])[8:], 20, 200, 64, True)])
def test_bytes_that_do_not_fit_are_refused(change):
    """(The kernels read as many bytes as the sizes say.)"""
    with pytest.raises(ValueError):
        GroupedWeight(*change(_weight().data))


def test_a_weights_bytes_are_not_exchanged():
    w = _weight()
    with pytest.raises(AttributeError):
        w.data = w.data.clone()
