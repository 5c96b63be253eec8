"""Which masks CrossAttention3d takes for a memory, and what it makes of them (no kernel is started here)."""
import copy
import pickle

import pytest
import torch
from torch.utils import _pytree

from d2conv3d_amd.attention import CrossAttention3d, Memory

cells = CrossAttention3d._cells


def memory(dims, N=2):
    T, H, W = dims
    k = torch.zeros(N, T * H * W, 2, 8)
    return Memory(k, k, dims)


def test_frames_and_cells():
    kept = memory((3, 6, 7))
    frames = torch.rand(2, 3) < 0.5
    want = frames[:, :, None].expand(2, 3, 42).reshape(2, 126)
    for mask in (frames, frames[:, :, None, None], want.view(2, 3, 6, 7), want):
        assert torch.equal(cells(mask, kept), want)
    key, value = kept                                   # (a pair as any other)
    assert torch.equal(cells(frames, (key, value)), want) and torch.equal(cells(want, [key, value]), want)
    one = torch.rand(2, 1) < 0.5
    assert torch.equal(cells(one, memory((1, 4, 5))), one.expand(2, 20))


@pytest.mark.parametrize("shape", [(2, 1), (2, 2), (2, 6), (2, 42), (2, 63), (2, 5), (2, 0), (2, 6, 3, 7), (2, 2, 3)])
def test_masks_of_another_number_of_frames_are_refused(shape):
    """... also where their width divides the number of cells"""
    with pytest.raises(RuntimeError, match="does not fit"):
        cells(torch.ones(shape, dtype=torch.bool), memory((3, 6, 7)))


def test_pairs_of_unknown_frames_take_what_divides():
    kept = tuple(memory((3, 6, 7)))
    assert cells(torch.ones(2, 2, dtype=torch.bool), kept).shape == (2, 126)
    with pytest.raises(RuntimeError, match="does not fit"):
        cells(torch.ones(2, 5, dtype=torch.bool), kept)


def test_no_cells():
    assert cells(torch.ones(2, 3, dtype=torch.bool), memory((3, 0, 5))).shape == (2, 0)
    assert cells(torch.ones(2, 0, dtype=torch.bool), memory((0, 4, 5))).shape == (2, 0)


def test_a_memory_is_a_pair_wherever_it_goes():
    kept = memory((3, 6, 7))
    leaves, spec = _pytree.tree_flatten((kept, 1))
    assert len(leaves) == 3
    for other in (copy.copy(kept), copy.deepcopy(kept), pickle.loads(pickle.dumps(kept)), _pytree.tree_unflatten(leaves, spec)[0]):
        assert type(other) is Memory and other.dims == (3, 6, 7) and len(other) == 2
        assert all(torch.equal(a, b) for a, b in zip(other, kept))
