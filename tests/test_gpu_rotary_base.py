"""rotary3d with bases that are no float32 numbers, and with positions beyond 2^24, against the definition in float64.  Bounds: test_gpu_rotary.py (2^-20 of a
pair's length to positions of 2^24); beyond, an angle is off by up to 2 pi 2^-48 of position * rate besides."""
import math

import pytest
import torch

import d2conv3d_amd as d2c
from d2conv3d_amd import attention
from d2conv3d_amd.attention import default_axis_pairs
from test_gpu_rotary import check, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("route", ["native", "python"])
@pytest.mark.parametrize("base", [10000.1, 10000.0 / 3.0, 499999.99, 1.1, math.pi])
def test_any_base(base, route, dev, monkeypatch):
    if route == "python":
        monkeypatch.setattr(attention, "_try_native", lambda *a: None)
    x = torch.randn(1, 60, 2, 40, generator=torch.Generator().manual_seed(2))
    pos = torch.randint(-(1 << 24), 1 << 24, (60, 3), generator=torch.Generator().manual_seed(3))
    xd = x.to(dev).requires_grad_()
    y = d2c.rotary3d(xd, pos.to(dev), base=base)
    check(y, reference(x, pos[:, None], default_axis_pairs(40), base, False), str(base))
    (gx,) = torch.autograd.grad(y, xd, x.to(dev))
    check(gx, reference(x, pos[:, None], default_axis_pairs(40), base, False, -1.0), str(base))


def test_positions_beyond_2_to_the_24(dev):
    x = torch.randn(1, 60, 2, 40, generator=torch.Generator().manual_seed(2))
    pos = torch.randint(-(1 << 30), 1 << 30, (60, 3), generator=torch.Generator().manual_seed(3)).float()
    e, b = reference(x, pos[:, None], default_axis_pairs(40), 10000.0, False)
    y = d2c.rotary3d(x.to(dev), pos.to(dev))
    far = 2 * math.pi * 2.0 ** -48 * 2.0 ** 30 / (2 * math.pi)          # (rates are below 1)
    length = (x[..., :20].double() ** 2 + x[..., 20:].double() ** 2).sqrt()
    check(y, (e, b + far * torch.cat([length, length], -1)))


def test_bases_that_are_refused(dev):
    x = torch.zeros(1, 6, 1, 8, device=dev)
    for base in (0.0, -1.0, math.inf, math.nan, 1e-60, 1e60):
        with pytest.raises(RuntimeError, match="base"):
            d2c.rotary3d(x, (1, 2, 3), base=base)
