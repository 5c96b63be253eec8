"""layer_norm against the definition in float64.

Bounds: u = 2^-8 (bfloat16) or 0 of the result for its one rounding, and float32 arithmetic: mean and variance are sums over C by lanes and a
tree, (C / 64 + 16) u32 relative to the mean magnitude of what is added up; the deviation x - mean so carries that
much of |x|.  A gradient of the parameters is a sum over the rows: (rows / 64 + 64) u32 of the magnitudes."""
import math

import pytest
import torch
import torch.nn as nn

import d2conv3d_amd as d2c

pytestmark = pytest.mark.gpu

U32, U16 = 2.0 ** -24, 2.0 ** -8


def make(shape, dtype, ptype, seed, mean=0.5, std=1.0):
    gen = torch.Generator().manual_seed(seed)
    C = shape[-1]

    def rn(*s):
        return torch.randn(*s, generator=gen)
    return ((rn(*shape) * std + mean).to(dtype), (rn(C) * 0.3 + 1).to(ptype), (rn(C) * 0.3).to(ptype), rn(*shape).to(dtype))


def reference(x, w, b, g, eps=1e-5):
    C = x.shape[-1]
    X, W, B, G = (t.double() for t in (x, w, b, g))
    mean = X.mean(-1, keepdim=True)
    std = ((X - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    h = (X - mean) / std
    y = h * W + B
    t = G * W
    gx = (t - t.mean(-1, keepdim=True) - h * (t * h).mean(-1, keepdim=True)) / std
    lead = tuple(range(x.dim() - 1))
    gw, gb = (G * h).sum(lead), G.sum(lead)
    u, up = (U16 if x.dtype == torch.bfloat16 else U32), (U16 if w.dtype == torch.bfloat16 else U32)
    e = (C / 64 + 16) * U32
    eh = e * (X.abs().mean(-1, keepdim=True) + X.abs()) / std + 2 * e * h.abs()
    rows = x.numel() // C
    er = (rows / 64 + 64) * U32
    t1, t2 = t.abs().mean(-1, keepdim=True), (t * h).abs().mean(-1, keepdim=True)
    et2 = (t.abs() * eh).mean(-1, keepdim=True) + e * t2
    bx = (4 * e * (t.abs() + t1 + h.abs() * t2) + eh * t2 + h.abs() * et2) / std + u * gx.abs()
    bounds = (eh * W.abs() + 2 * U32 * (h * W).abs() + 2 * U32 * B.abs() + u * y.abs(), bx,
              (G.abs() * eh).sum(lead) + er * (G * h).abs().sum(lead) + up * gw.abs(), er * G.abs().sum(lead) + up * gb.abs())
    return (y, gx, gw, gb), bounds


def check(got, want, bounds, what=""):
    for name, a, e, b in zip(("out", "grad_input", "grad_weight", "grad_bias"), got, want, bounds):
        a = a.detach().double().cpu()
        assert a.shape == e.shape
        over = (a - e).abs() / (1.05 * b + 1e-30)
        assert not bool((~(over <= 1.0)).any()), f"{what} {name}: worst {over.max().item():.2f} of the bound, NaN {int(a.isnan().sum())}"


def run(dev, x, w, b, g, eps=1e-5):
    args = [t.to(dev).requires_grad_() for t in (x, w, b)]
    out = d2c.layer_norm(*args, eps=eps)
    grads = torch.autograd.grad(out, args, g.to(dev))
    torch.cuda.synchronize(dev)
    return (out, *grads)


SHAPES = [(1, 1), (3, 2), (5, 7), (2, 9, 64), (70, 65), (33, 128), (9, 250), (40, 257), (300, 512), (17, 1000), (5, 2048), (4, 2049),
          (3, 4100), (2, 8192), (3, 8200), (2, 16384), (5000, 96), (1, 16), (2, 700, 24)]


@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_gradients(shape, types, dev):
    print("layer_norm", shape, types, flush=True)
    x, w, b, g = make(shape, *types, seed=sum(shape))
    want, bounds = reference(x, w, b, g)
    got = run(dev, x, w, b, g)
    check(got, want, bounds, str(shape))
    for a, c in zip(got, run(dev, x, w, b, g)):
        assert torch.equal(a, c)
    with torch.no_grad():
        assert torch.equal(d2c.layer_norm(x.to(dev), w.to(dev), b.to(dev)), got[0])


def test_a_mean_far_above_the_spread(dev):
    """Deviations are taken from the mean itself: mean 1000, spread 0.5."""
    x, w, b, g = make((50, 512), torch.float32, torch.float32, 3, 1000.0, 0.5)
    want, bounds = reference(x, w, b, g)
    check(run(dev, x, w, b, g), want, bounds)


def test_constant_rows(dev):
    x = torch.full((4, 100), 3.25)
    _, w, b, g = make((4, 100), torch.float32, torch.float32, 3)
    out = run(dev, x, w, b, g)[0]
    assert torch.equal(out.cpu(), b.expand(4, 100))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_anywhere(dtype, dev):
    x, w, b, g = make((2, 30, 100), dtype, dtype, 11)
    want, bounds = reference(x, w, b, g)
    buf = torch.full((2, 30, 307), math.nan, dtype=dtype, device=dev)
    buf[..., 101:201] = x.to(dev)
    views = {"part of a wider row": buf[..., 101:201],
             "channels first": x.to(dev).transpose(1, 2).contiguous().transpose(1, 2),
             "positions first": x.to(dev).transpose(0, 1).contiguous().transpose(0, 1)}
    for how, xd in views.items():
        args = [xd.requires_grad_(), w.to(dev).requires_grad_(), b.to(dev).requires_grad_()]
        gd = g.to(dev).transpose(1, 2).contiguous().transpose(1, 2)
        out = d2c.layer_norm(*args)
        check((out, *torch.autograd.grad(out, args, gd)), want, bounds, how)


def test_without_parameters_and_some_gradients(dev):
    x, w, b, g = make((40, 200), torch.float32, torch.float32, 13)
    one, zero = torch.ones(200), torch.zeros(200)
    for weight, bias in ((None, None), (w, None), (None, b)):
        want, bounds = reference(x, one if weight is None else w, zero if bias is None else b, g)
        args = [None if t is None else t.to(dev).requires_grad_() for t in (x, weight, bias)]
        out = d2c.layer_norm(*args)
        grads = iter(torch.autograd.grad(out, [t for t in args if t is not None], g.to(dev)))
        got = (out, *(next(grads) if t is not None else None for t in args))
        sel = [i for i, t in enumerate(got) if t is not None]
        check([got[i] for i in sel], [want[i] for i in sel], [bounds[i] for i in sel])
    want, bounds = reference(x, w, b, g)
    wd = w.to(dev).requires_grad_()
    (gw,) = torch.autograd.grad(d2c.layer_norm(x.to(dev), wd, b.to(dev)), wd, g.to(dev))
    check((gw,), (want[2],), (bounds[2],))


def test_no_rows(dev):
    x = torch.zeros(0, 50, device=dev, requires_grad=True)
    w, b = torch.ones(50, device=dev, requires_grad=True), torch.zeros(50, device=dev, requires_grad=True)
    out = d2c.layer_norm(x, w, b)
    gx, gw, gb = torch.autograd.grad(out, (x, w, b), torch.zeros_like(out))
    assert out.shape == (0, 50) and gx.shape == (0, 50) and not bool(gw.any()) and not bool(gb.any())


def test_gradients_against_differences(dev):
    x, w, b, g = (t.to(dev) for t in make((20, 130), torch.float32, torch.float32, 17))
    ts = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(d2c.layer_norm(*ts), ts, g)
    h, gen = 2.0 ** -7, torch.Generator(device=dev).manual_seed(5)
    for i in range(3):
        step = torch.randn(ts[i].shape, generator=gen, device=dev)

        def loss(sign):
            args = [t.detach() + (sign * h * step if j == i else 0) for j, t in enumerate(ts)]
            return (d2c.layer_norm(*args).double() * g.double()).sum()
        slope, exact = ((loss(1) - loss(-1)) / (2 * h)).item(), (grads[i].double() * step.double()).sum().item()
        size = (grads[i].double() * step.double()).norm().item()
        assert abs(slope - exact) <= 5e-3 * max(size, abs(exact)), (i, slope, exact)


def test_float16_and_module(dev):
    x, w, b, g = make((30, 64), torch.float16, torch.float16, 19)
    want, bounds = reference(x.float(), w.float(), b.float(), g.float())
    got = run(dev, x, w, b, g)
    assert all(t.dtype == torch.float16 for t in got)
    check(got, want, [v + 2.0 ** -11 * e.abs() + 2.0 ** -24 for v, e in zip(bounds, want)])
    m = d2c.LayerNorm(64).to(dev)
    assert isinstance(m, nn.LayerNorm) and set(m.state_dict()) == {"weight", "bias"}
    xf = x.float().to(dev)
    assert torch.equal(m(xf), d2c.layer_norm(xf, m.weight, m.bias))


def test_more_rows_than_2_to_the_31_elements_reach(dev):
    """Rows so far apart that the last starts beyond 2^31 elements."""
    rows, C = 70, 40
    gap = (1 << 31) // (rows - 1) + 1
    x, w, b, g = make((rows, C), torch.bfloat16, torch.float32, 23)
    buf = torch.empty(gap * rows, dtype=torch.bfloat16, device=dev)
    xd = torch.as_strided(buf, (rows, C), (gap, 1))
    xd.copy_(x.to(dev))
    want, bounds = reference(x, w, b, g)
    args = [xd.requires_grad_(), w.to(dev).requires_grad_(), b.to(dev).requires_grad_()]
    out = d2c.layer_norm(*args)
    check((out, *torch.autograd.grad(out, args, g.to(dev))), want, bounds)


def test_refusals(dev):
    x, w, b, _ = (t.to(dev) for t in make((4, 32), torch.float32, torch.float32, 1))
    for args, text in (((x, w[:31], b), "weight must have the shape"), ((x, w, b[None]), "bias must have the shape"),
                       ((x.cpu(), w, b), "on the GPU"), ((x, w.cpu(), b), "on the GPU"), ((x.double(), w.double(), b.double()), "unsupported dtype"),
                       ((x[:, :0], None, None), "last dimension"), ((torch.zeros(2, 16385, device=dev),), "up to 16384")):
        with pytest.raises(RuntimeError, match=text):
            d2c.layer_norm(*args)
    with pytest.raises(RuntimeError, match="eps"):
        d2c.layer_norm(x, w, b, eps=-1.0)
