"""CrossAttention3d without samples, without positions and without a memory's cells: results and gradients of the shapes that they would have."""
import pytest
import torch

import d2conv3d_amd as d2c

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,dims,other", [(0, (2, 3, 4), (1, 3, 4)), (2, (0, 3, 4), (1, 3, 4)), (2, (2, 3, 4), (0, 3, 4)), (0, (0, 3, 4), (0, 3, 4))])
def test_nothing(N, dims, other, dtype, dev):
    block = d2c.CrossAttention3d(32, heads=2, kv_heads=1).to(dev, dtype)
    for p in block.out.parameters():
        torch.nn.init.normal_(p)
    x = torch.randn(N, 32, *dims, device=dev, dtype=dtype, requires_grad=True)
    memory = torch.randn(N, 32, *other, device=dev, dtype=dtype, requires_grad=True)
    for mask in (None, torch.ones(N, other[0], dtype=torch.bool, device=dev)):
        out = block(x, memory, memory_mask=mask)
        assert out.shape == x.shape
        gx, gm = torch.autograd.grad(out, (x, memory), torch.ones_like(out))
        assert gx.shape == x.shape and gm.shape == memory.shape
        with torch.no_grad():
            assert torch.equal(block(x, block.remember(memory), memory_mask=mask), out)
        if other[0] == 0:
            assert torch.equal(out, x + block.out.bias.view(-1, 1, 1, 1))
