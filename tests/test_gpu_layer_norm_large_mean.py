"""layer_norm of rows that are constant and so large that mean * rstd leaves float32's range: deviations are 0, outputs the bias, gradients those of the
definition (rstd (g w - mean(g w))), whatever the row's length; nothing behind a row's end counts.  Bound of the gradient: float32 sums over C channels."""
import pytest
import torch

import d2conv3d_amd as d2c

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("C", [3, 9, 33, 64, 100, 120])
def test_large_constant_rows(C, dtype, dev):
    gen = torch.Generator().manual_seed(C)
    x = torch.tensor([2.0 ** 120, -(2.0 ** 120), 2.0 ** 119, 1.0])[:, None].expand(4, C).to(dtype)
    w, b, g = torch.randn(C, generator=gen), torch.randn(C, generator=gen), torch.randn(4, C, generator=gen).to(dtype)
    args = [t.to(dev).requires_grad_() for t in (x, w, b)]
    out = d2c.layer_norm(*args)
    gx, gw, gb = (t.double().cpu() for t in torch.autograd.grad(out, args, g.to(dev)))
    assert torch.equal(out.cpu(), b.to(dtype).expand(4, C))
    u = g.double() * w.double()
    want = (u - u.mean(1, keepdim=True)) / 1e-5 ** 0.5
    bound = 2.0 ** -24 * (C + 16) * (u.abs() + u.abs().mean(1, keepdim=True)) / 1e-5 ** 0.5 + (2.0 ** -8 if dtype == torch.bfloat16 else 0) * want.abs()
    assert bool(((gx - want).abs() <= bound).all()), ((gx - want).abs() / bound).max()
    assert not bool(gw.any())
    assert bool(((gb - g.double().sum(0)).abs() <= 2.0 ** -22 * g.double().abs().sum(0)).all())
