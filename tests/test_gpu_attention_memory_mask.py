"""CrossAttention3d refuses a mask of a number of frames that its memory does not have, as a map or kept."""
import pytest
import torch

import d2conv3d_amd as d2c

pytestmark = pytest.mark.gpu


def test_a_mask_of_other_frames(dev):
    block = d2c.CrossAttention3d(32, heads=2).to(dev)
    torch.nn.init.normal_(block.out.weight)
    x, memory = torch.randn(1, 32, 1, 2, 2, device=dev), torch.randn(1, 32, 3, 4, 2, device=dev)
    with torch.no_grad():
        kept = block.remember(memory)
        assert len(kept) == 2 and kept.dims == (3, 4, 2)
        for m in (memory, kept):
            for frames in (2, 4, 6, 8, 12):
                with pytest.raises(RuntimeError, match="does not fit"):
                    block(x, m, memory_mask=torch.ones(1, frames, dtype=torch.bool, device=dev))
            keep = torch.tensor([[True, False, True]], device=dev)
            want = block(x, memory[:, :, [0, 2]], memory_positions=torch.cartesian_prod(
                torch.tensor([0, 2], device=dev), torch.arange(4, device=dev), torch.arange(2, device=dev)))
            assert torch.allclose(block(x, m, memory_mask=keep), want, rtol=1e-5, atol=1e-5)
