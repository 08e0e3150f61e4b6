"""Calls of cache.reorder that are refused leave every tensor as it was."""
import pytest
import torch

from w8a8 import W8A8Error, cache

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_a_tensor_too_large_is_refused_before_any_is_reordered():
    """More tensors than one launch takes, the last with more columns than the kernel counts (rows of over 2 GiB at an odd
    address)."""
    g = torch.Generator(device=DEV).manual_seed(1)
    small = [torch.randn(2, 40, generator=g, device=DEV) for _ in range(48)]
    want = [t.clone() for t in small]
    row = (1 << 31) + 3
    large = torch.zeros(2 * row + 1, dtype=torch.int8, device=DEV)[1:].view(2, row)
    large[1, -1] = 5
    with pytest.raises(W8A8Error, match="tensor 48 too large"):
        cache.reorder([*small, large], torch.tensor([1, 1], device=DEV))
    assert all(torch.equal(t, w) for t, w in zip(small, want))
    assert large[:, -1].tolist() == [0, 5]


def test_the_index_among_the_tensors_is_refused():
    """The beams' numbers kept beside their states: a copy of the index reorders them too."""
    t, beams = torch.arange(12, device=DEV).view(4, 3).clone(), torch.tensor([1, 2, 3, 0], device=DEV)
    with pytest.raises(W8A8Error, match="index lies in tensor 1"):
        cache.reorder([t, beams], beams)
    assert t.flatten().tolist() == list(range(12)) and beams.tolist() == [1, 2, 3, 0]
    cache.reorder([t, beams], beams.clone())
    assert t[:, 0].tolist() == [3, 6, 9, 0] and beams.tolist() == [2, 3, 0, 1]
