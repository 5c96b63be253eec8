"""rotary3d against the definition in float64, element by element.

Bounds: an angle is exact to float32 (an error of 2^-23 turns, 2 pi 2^-23 radians, and the cosine's own 2^-22), so a turned value is off by 2^-20 of
the pair's length, and once rounded: 2^-8 of its size in bfloat16, 2^-24 in float32."""
import math

import pytest
import torch

import d2conv3d_amd as d2c
from d2conv3d_amd.attention import default_axis_pairs

pytestmark = pytest.mark.gpu


def reference(x, pos, pairs, base, interleaved, sign=1.0):
    """(y, bound) in float64; pos [L, 3] or [N, L, 3]"""
    X, pos = x.double(), pos.double()
    y, bound = X.clone(), torch.zeros_like(X)
    j, total = 0, sum(pairs)
    for axis in range(3):
        for i in range(pairs[axis]):
            a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + total)
            angle = sign * pos[..., axis] * float(base) ** (-i / pairs[axis])
            c, s = torch.cos(angle), torch.sin(angle)
            y[..., a], y[..., b] = X[..., a] * c - X[..., b] * s, X[..., a] * s + X[..., b] * c
            length = (X[..., a] ** 2 + X[..., b] ** 2).sqrt()
            bound[..., a] = bound[..., b] = 2.0 ** -20 * length
            j += 1
    u = 2.0 ** -8 if x.dtype == torch.bfloat16 else 2.0 ** -24
    return y, bound + u * y.abs()


def grid_positions(T, H, W):
    i = torch.arange(T * H * W)
    return torch.stack([i // (H * W), i // W % H, i % W], -1)


def check(a, want, what=""):
    e, b = want
    a = a.detach().double().cpu()
    assert a.shape == e.shape
    over = (a - e).abs() / (1.05 * b + 1e-30)
    assert not bool((~(over <= 1.0)).any()), f"{what}: worst {over.max().item():.2f} of the bound, NaN {int(a.isnan().sum())}"


CASES = [
    # N, grid, heads, D, pairs
    (1, (1, 1, 1), 1, 2, (1, 0, 0)),
    (2, (3, 4, 5), 2, 64, None),
    (1, (1, 14, 25), 8, 64, None),
    (2, (2, 7, 9), 3, 40, None),
    (1, (5, 3, 2), 1, 24, None),
    (3, (2, 3, 5), 4, 33, (3, 4, 5)),
    (1, (4, 6, 7), 2, 128, (16, 24, 24)),
    (1, (2, 5, 6), 2, 80, (0, 20, 20)),
    (2, (1, 3, 11), 5, 7, (1, 1, 1)),
    (1, (2, 2, 2), 2, 20, (0, 0, 0)),
    (1, (3, 3, 3), 1, 256, (43, 43, 42)),
    (1, (8, 30, 31), 6, 96, None),
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", CASES)
def test_forward_and_gradient(case, dtype, interleaved, dev):
    print("rotary3d", case, dtype, interleaved, flush=True)
    N, grid, heads, D, pairs = case
    gen = torch.Generator().manual_seed(D + heads)
    L = math.prod(grid)
    x, g = (torch.randn(N, L, heads, D, generator=gen).to(dtype) for _ in range(2))
    real = torch.rand(N, L, 3, generator=gen) * 300 - 100
    used = default_axis_pairs(D) if pairs is None else pairs
    for positions, pos in ((grid, grid_positions(*grid)), (real.to(dev), real), (real[0].to(dev), real[0]),
                           ((real[0] * 1000).long().to(dev), (real[0] * 1000).long())):
        xd = x.to(dev).requires_grad_()
        y = d2c.rotary3d(xd, positions, pairs, interleaved=interleaved)
        (gx,) = torch.autograd.grad(y, xd, g.to(dev))
        for i, (got, src, sign) in enumerate(((y, x, 1.0), (gx, g, -1.0))):
            e, b = reference(src, pos[..., None, :] if pos.dim() == 2 else pos[:, :, None], used, 10000.0, interleaved, sign)
            check(got, (e, b), f"{case} {i}")


def test_far_positions_and_bases(dev):
    x = torch.randn(1, 50, 2, 32, generator=torch.Generator().manual_seed(2))
    pos = torch.randint(-(1 << 24), 1 << 24, (50, 3), generator=torch.Generator().manual_seed(3))
    for base in (10000.0, 500000.0, 10.0, 1.0):
        y = d2c.rotary3d(x.to(dev), pos.to(dev), base=base)
        check(y, reference(x, pos[:, None], default_axis_pairs(32), base, False), str(base))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(dtype, dev):
    N, grid, heads, D = 2, (2, 3, 7), 3, 40
    gen = torch.Generator().manual_seed(7)
    x, g = (torch.randn(N, 42, heads, D, generator=gen).to(dtype) for _ in range(2))
    want = reference(x, grid_positions(*grid)[:, None], default_axis_pairs(D), 1e4, False)
    back = reference(g, grid_positions(*grid)[:, None], default_axis_pairs(D), 1e4, False, -1.0)

    def views(t):
        t = t.to(dev)
        buf = torch.full((N, 42, 2, heads, D + 1), math.nan, dtype=dtype, device=dev)
        buf[:, :, 1, :, 1:] = t
        return {"part of a projection": buf[:, :, 1, :, 1:],
                "heads first": t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3),
                "channels apart": t.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2)}
    for (how, xd), gd in zip(views(x).items(), views(g).values()):
        xd.requires_grad_()
        y = d2c.rotary3d(xd, grid)
        check(y, want, how)
        check(torch.autograd.grad(y, xd, gd)[0], back, how)


def test_gradient_against_differences(dev):
    gen = torch.Generator(device=dev).manual_seed(11)
    x, g, step = (torch.randn(1, 30, 2, 24, generator=gen, device=dev) for _ in range(3))
    pos = torch.rand(30, 3, generator=gen, device=dev) * 50
    x.requires_grad_()
    (gx,) = torch.autograd.grad(d2c.rotary3d(x, pos, interleaved=True), x, g)

    def loss(s):
        return (d2c.rotary3d(x.detach() + s * step, pos, interleaved=True).double() * g.double()).sum()
    slope, exact = ((loss(0.5) - loss(-0.5)) / 1.0).item(), (gx.double() * step.double()).sum().item()
    assert abs(slope - exact) <= 1e-4 * (gx.double() * step.double()).norm().item()      # (linear in x)


def test_nothing_to_turn_and_float16(dev):
    assert d2c.rotary3d(torch.zeros(0, 6, 2, 8, device=dev), (1, 2, 3)).shape == (0, 6, 2, 8)
    assert d2c.rotary3d(torch.zeros(2, 0, 2, 8, device=dev), torch.zeros(0, 3, device=dev)).shape == (2, 0, 2, 8)
    x = torch.randn(1, 12, 2, 16, generator=torch.Generator().manual_seed(1)).half()
    y = d2c.rotary3d(x.to(dev), (1, 3, 4))
    e, b = reference(x.float(), grid_positions(1, 3, 4)[:, None], default_axis_pairs(16), 1e4, False)
    assert y.dtype == torch.float16
    check(y, (e, b + 2.0 ** -11 * e.abs() + 2.0 ** -24))


def test_refusals(dev):
    x = torch.zeros(2, 12, 2, 16, device=dev)
    for args, kw, text in (((x[0], (1, 3, 4)), {}, "input must be"), ((x, (1, 3, 5)), {}, "is not 12 tokens"),
                           ((x, torch.zeros(12, 2, device=dev)), {}, "positions must be"), ((x, torch.zeros(3, 12, 3, device=dev)), {}, "positions must be"),
                           ((x, torch.zeros(12, 3)), {}, "on the GPU"), ((x, torch.zeros(12, 3, device=dev, requires_grad=True)), {}, "no gradient"),
                           ((x, (1, 3, 4), (4, 4, 1)), {}, "do not fit"), ((x, (1, 3, 4), (4, 4)), {}, "axis_pairs"),
                           ((x, (1, 3, 4), (-1, 4, 1)), {}, "axis_pairs"), ((x.double(), (1, 3, 4)), {}, "unsupported dtype"),
                           ((x.cpu(), (1, 3, 4)), {}, "on the GPU"), ((x, (1, 3, 4)), dict(base=0.0), "base")):
        with pytest.raises(RuntimeError, match=text):
            d2c.rotary3d(*args, **kw)
    wide = torch.zeros(1, 1, 1, 300, device=dev)
    with pytest.raises(RuntimeError, match="up to 128 pairs"):
        d2c.rotary3d(wide, (1, 1, 1), (50, 50, 50))
