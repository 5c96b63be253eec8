"""cross_attention against the definition in float64, forward and all gradients, element by element.

Bounds (u = the unit roundoff, 2^-8 for bfloat16 and 2^-24 for float32; A = sum_j p_j |v_j| and its like for the gradients):
bfloat16 rounds the weights p (and ds) to the matrix instruction's operands and the result once, u each, so an output is off by 2 u A; a
gradient through the scores also carries delta = sum_d do o, made of the rounded output.  What float32 arithmetic adds is bounded
by E = u32 (D + 64 + L / 8 + 4 max_s) A, L the length of the sum: products and sums over D channels and L positions on the matrix
instruction, and an exponential whose argument of size max_s is rounded."""
import math

import pytest
import torch

import d2conv3d_amd as d2c
from _util import assert_close

pytestmark = pytest.mark.gpu

U32, U16 = 2.0 ** -24, 2.0 ** -8


def make(N, Lq, Lk, Hq, Hkv, D, dtype, seed, std=1.0):
    gen = torch.Generator().manual_seed(seed)

    def rn(*shape, s=1.0):
        return (torch.randn(*shape, generator=gen) * s).to(dtype)
    return rn(N, Lq, Hq, D, s=std), rn(N, Lk, Hkv, D), rn(N, Lk, Hkv, D), rn(N, Lq, Hq, D)


def make_masks(kind, N, Lk, seed):
    gen = torch.Generator().manual_seed(seed + 1)
    lengths = mask = None
    if kind in ("lengths", "both"):
        lengths = torch.randint(0, Lk + 1, (N,), generator=gen)
        lengths[0] = 0                       # a sample without keys
        if N > 1:
            lengths[1] = Lk
    if kind in ("mask", "both"):
        mask = torch.rand(N, Lk, generator=gen) < 0.6
        if N > 1:
            mask[1] = False                  # ... and another way to have none
    return lengths, mask


def reference(q, k, v, g, lengths, mask, scale):
    """(out, gq, gk, gv) in float64 and for each the bound of the type's errors."""
    dtype = q.dtype
    u = U16 if dtype == torch.bfloat16 else 0.0
    N, Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[1:3]
    ok = torch.ones(N, Lk, dtype=torch.bool)
    if lengths is not None:
        ok &= torch.arange(Lk) < lengths[:, None]
    if mask is not None:
        ok &= mask
    rep = Hq // Hkv
    Q, G = (t.double().permute(0, 2, 1, 3).contiguous() for t in (q, g))
    K, V = (torch.where(ok[:, :, None, None], t.double(), 0.0).permute(0, 2, 1, 3).repeat_interleave(rep, 1).contiguous()
            for t in (k, v))

    def shared(t):      # [N, Hq, Lk, D] -> [N, Lk, Hkv, D]
        return t.view(N, Hkv, rep, Lk, D).sum(2).permute(0, 2, 1, 3)

    def heads_last(t):
        return t.permute(0, 2, 1, 3)
    allowed = ok[:, None, None, :]
    s = (Q @ K.transpose(-1, -2)) * scale
    sabs = (Q.abs() @ K.abs().transpose(-1, -2)) * scale
    s = s.masked_fill(~allowed, -math.inf)
    top = s.amax(-1, keepdim=True) if Lk else torch.full((N, Hq, Lq, 1), -math.inf, dtype=torch.float64)
    e = torch.exp(s - torch.where(top.isinf(), 0.0, top))
    p = e / e.sum(-1, keepdim=True).clamp_min(1e-300)
    out = p @ V
    gp = G @ V.transpose(-1, -2)
    delta = (G * out).sum(-1, keepdim=True)
    ds = p * (gp - delta)
    gq, gk, gv = ds @ K * scale, ds.transpose(-1, -2) @ Q * scale, p.transpose(-1, -2) @ G
    smax = sabs.max().item() if sabs.numel() else 0.0
    e32 = U32 * (D + 64 + max(Lq * rep, Lk) / 8 + 4 * smax)
    A = p @ V.abs()
    b_out = (2 * u + 2 * e32) * A
    pabs = p * (G.abs() @ V.abs().transpose(-1, -2) + (G.abs() * A).sum(-1, keepdim=True))
    ddelta = (G.abs() * b_out).sum(-1, keepdim=True)
    eds = u * ds.abs() + p * ddelta + 4 * e32 * pabs
    b_q = (eds @ K.abs() + 2 * e32 * (pabs @ K.abs())) * scale + u * gq.abs()
    b_k = (eds.transpose(-1, -2) @ Q.abs() + 2 * e32 * (pabs.transpose(-1, -2) @ Q.abs())) * scale
    b_v = (u + 2 * e32) * (p.transpose(-1, -2) @ G.abs())
    gk, gv, b_k, b_v = shared(gk), shared(gv), shared(b_k), shared(b_v)
    return ((heads_last(out), heads_last(gq), gk, gv),
            (heads_last(b_out), heads_last(b_q), b_k + u * gk.abs(), b_v + u * gv.abs()))


def check(got, want, bounds, what=""):
    for name, a, e, b in zip(("out", "grad_query", "grad_key", "grad_value"), got, want, bounds):
        a = a.detach().double().cpu()
        assert a.shape == e.shape, (what, name, a.shape, e.shape)
        bound = 1.05 * b + 1e-30
        over = (a - e).abs() / bound
        assert not bool((~(over <= 1.0)).any()), (
            f"{what} {name}: {int((~(over <= 1.0)).sum())} of {over.numel()} beyond the bound, worst {over.max().item():.2f} of it, "
            f"NaN {int(a.isnan().sum())}")


def run(dev, q, k, v, g, lengths, mask, scale=None):
    args = [t.to(dev).requires_grad_() for t in (q, k, v)]
    out = d2c.cross_attention(*args, key_lengths=None if lengths is None else lengths.to(dev),
                              key_mask=None if mask is None else mask.to(dev), scale=scale)
    grads = torch.autograd.grad(out, args, g.to(dev))
    torch.cuda.synchronize(dev)
    return (out, *grads)


CASES = [
    # N, Lq, Lk, Hq, Hkv, D, mask
    (1, 1, 1, 1, 1, 64, "none"),
    (2, 1, 5, 4, 1, 32, "none"),
    (1, 3, 64, 2, 2, 64, "none"),
    (2, 33, 65, 4, 2, 40, "none"),
    (1, 128, 128, 2, 1, 128, "none"),
    (1, 129, 127, 1, 1, 96, "mask"),
    (3, 7, 300, 6, 2, 24, "lengths"),
    (2, 50, 200, 4, 4, 72, "mask"),
    (3, 16, 1000, 8, 1, 80, "both"),
    (1, 9, 31, 2, 2, 1, "none"),
    (2, 20, 70, 3, 1, 7, "lengths"),
    (1, 65, 33, 2, 2, 33, "none"),
    (2, 40, 100, 2, 1, 100, "both"),
    (1, 31, 129, 1, 1, 127, "mask"),
    (1, 1, 4000, 2, 1, 128, "none"),        # one row, keys shared by workgroups
    (1, 40, 3000, 1, 1, 64, "mask"),
    (2, 1500, 40, 2, 1, 64, "lengths"),     # few keys, rows shared by workgroups
    (1, 300, 700, 12, 3, 32, "both"),
    (2, 70, 150, 2, 1, 104, "lengths"),     # heads that fill the widest kernels in part, in whole pieces of 16 bytes
    (1, 40, 260, 2, 2, 120, "mask"),
    (1, 130, 90, 3, 1, 88, "none"),
    (1, 20, 50, 1, 1, 8, "none"),
    (1, 50, 140, 2, 1, 16, "none"),
    (2, 1, 700, 8, 1, 64, "both"),          # up to 8 rows of a key head: one, two, four, eight, some not there
    (1, 2, 333, 4, 1, 40, "mask"),
    (3, 1, 1300, 6, 2, 96, "lengths"),
    (1, 1, 900, 1, 1, 7, "mask"),
    (1, 4, 257, 2, 1, 33, "none"),
    (2, 2, 64, 1, 1, 128, "lengths"),
    (1, 5, 2000, 1, 1, 24, "mask"),
    (1, 526, 984, 8, 8, 128, "none"),       # the widest heads, tiles that end inside and walks that are shared
    (2, 300, 1000, 4, 2, 104, "both"),
    (1, 150, 1100, 3, 1, 64, "mask"),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("case", CASES)
def test_forward_and_gradients(case, dtype, dev):
    print("cross_attention", case, dtype, flush=True)
    *sizes, kind = case
    q, k, v, g = make(*sizes, dtype, seed=sum(sizes))
    lengths, mask = make_masks(kind, sizes[0], sizes[2], sum(sizes))
    want, bounds = reference(q, k, v, g, lengths, mask, 1.0 / math.sqrt(sizes[-1]))
    got = run(dev, q, k, v, g, lengths, mask)
    check(got, want, bounds, str(case))
    again = run(dev, q, k, v, g, lengths, mask)
    for a, b in zip(got, again):
        assert torch.equal(a, b)             # sums in one order
    with torch.no_grad():
        alone = d2c.cross_attention(q.to(dev), k.to(dev), v.to(dev), None if lengths is None else lengths.to(dev),
                                    None if mask is None else mask.to(dev))
    assert torch.equal(alone, got[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("std,scale", [(12.0, None), (1.0, 3.0), (1.0, 1e-3)])
def test_scores_of_any_size(std, scale, dtype, dev):
    q, k, v, g = make(2, 37, 150, 2, 1, 64, dtype, 5, std)
    want, bounds = reference(q, k, v, g, None, None, 1.0 / 8 if scale is None else scale)
    check(run(dev, q, k, v, g, None, None, scale), want, bounds, f"{std} {scale}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Lq", [1, 70])
@pytest.mark.parametrize("garbage", [math.nan, math.inf, -math.inf, "lowest"])
def test_what_is_not_read_has_no_influence(garbage, Lq, dtype, dev):
    N, Lk = 3, 400
    q, k, v, g = make(N, Lq, Lk, 4, 2, 64, dtype, 9)
    lengths, mask = make_masks("both", N, Lk, 9)
    lengths[0], mask[0, :100] = 300, False
    want, bounds = reference(q, k, v, g, lengths, mask, 1.0 / 8)
    hidden = ~(mask & (torch.arange(Lk) < lengths[:, None]))
    value = torch.finfo(dtype).min if garbage == "lowest" else garbage
    k[hidden], v[hidden] = value, value
    got = run(dev, q, k, v, g, lengths, mask)
    check(got, want, bounds, str(garbage))
    assert not bool(got[0][1].any()) and not bool(got[1][1].any())      # the sample without keys
    assert not bool(got[2].cpu()[hidden].any()) and not bool(got[3].cpu()[hidden].any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(dtype, dev):
    N, Lq, Lk, Hq, Hkv, D = 2, 45, 90, 4, 2, 40
    q, k, v, g = make(N, Lq, Lk, Hq, Hkv, D, dtype, 21)
    want, bounds = reference(q, k, v, g, None, None, 1.0 / math.sqrt(D))

    def view(t, how):
        t = t.to(dev)
        n, l, h, d = t.shape
        if how == "heads first":
            return t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
        if how == "odd start":
            buf = torch.full((n, l, h, d + 3), math.nan, dtype=dtype, device=dev)
            buf[..., 1:d + 1] = t
            return buf[..., 1:d + 1]
        if how == "channels apart":
            return t.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2)
        if how == "backwards":
            return t.flip(1).contiguous().flip(1)
        buf = torch.full((n, l, 3, h, d), math.nan, dtype=dtype, device=dev)      # "projection"
        buf[:, :, 1] = t
        return buf[:, :, 1]
    for how in ("heads first", "odd start", "channels apart", "projection", "backwards"):
        args = [view(t, how).requires_grad_() for t in (q, k, v)]
        out = d2c.cross_attention(*args)
        grads = torch.autograd.grad(out, args, view(g, how))
        check((out, *grads), want, bounds, how)


def outputs_of(args, g, lengths, mask):
    out = d2c.cross_attention(*args, key_lengths=lengths, key_mask=mask)
    return (out, *torch.autograd.grad(out, args, g))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [8, 20, 24, 33, 40, 64, 70, 72, 80, 96, 100, 104, 120, 128])
def test_nothing_behind_the_tensors_is_read(D, dtype, dev):
    """Ends inside a tile, walks shared by workgroups, keys that are not to be read among those that are: what lies behind the
    last row of an input, or between its heads and rows, changes nothing."""
    print("cross_attention: NaN around the inputs", D, dtype, flush=True)
    for N, Lq, Lk, Hq, Hkv, kind in ((1, 526, 984, 8, 8, "none"), (2, 300, 2000, 4, 2, "both"), (3, 4, 1900, 3, 3, "lengths"),
                                     (1, 1500, 130, 2, 2, "none"), (1, 33, 700, 6, 2, "mask"), (2, 2, 400, 2, 2, "mask")):
        plain = make(N, Lq, Lk, Hq, Hkv, D, dtype, 91 + D)
        lengths, mask = make_masks(kind, N, Lk, 91)
        lengths, mask = (None if t is None else t.to(dev) for t in (lengths, mask))

        def inside(t, rows, gap):       # a part of a buffer of NaN
            n, l, h, d = t.shape
            buf = torch.full((n, l + rows, h, d + gap), math.nan, dtype=dtype, device=dev)
            buf[:, :l, :, :d] = t.to(dev)
            return buf[:, :l, :, :d]
        want = outputs_of([t.to(dev).requires_grad_() for t in plain[:3]], plain[3].to(dev), lengths, mask)
        assert not any(bool(t.isnan().any()) for t in want)
        for rows, gap in ((200, 0), (0, 8)):
            args = [inside(t, rows, gap).requires_grad_() for t in plain[:3]]
            for _ in range(3):
                got = outputs_of(args, inside(plain[3], rows, gap), lengths, mask)
                for a, b in zip(got, want):
                    assert torch.equal(a, b), (N, Lq, Lk, Hq, Hkv, kind, rows, gap)


def test_shared_and_broadcast_inputs(dev):
    """One memory for all samples (expanded), and one tensor as keys and values: gradients add up."""
    q, k, v, g = make(3, 20, 60, 4, 2, 32, torch.float32, 33)
    k = k[:1]
    kk = k.expand(3, -1, -1, -1)
    want, bounds = reference(q, kk, kk, g, None, None, 1.0 / math.sqrt(32))
    qd, kd = q.to(dev).requires_grad_(), k.to(dev).requires_grad_()
    e = kd.expand(3, -1, -1, -1)
    out = d2c.cross_attention(qd, e, e)
    gq, gk = torch.autograd.grad(out, (qd, kd), g.to(dev))
    check((out, gq), want[:2], bounds[:2])
    both = (want[2] + want[3]).sum(0, keepdim=True)
    bound = (bounds[2] + bounds[3]).sum(0, keepdim=True) + 4 * U32 * (want[2].abs() + want[3].abs()).sum(0, keepdim=True)
    assert bool(((gk.double().cpu() - both).abs() <= 1.05 * bound).all())


@pytest.mark.parametrize("Lq,Lk", [(0, 5), (5, 0), (0, 0)])
def test_no_rows_or_no_keys(Lq, Lk, dev):
    for dtype in (torch.float32, torch.bfloat16):
        q, k, v, g = make(2, Lq, Lk, 3, 1, 7, dtype, 3)
        out, gq, gk, gv = run(dev, q, k, v, g, None, None)
        assert out.shape == q.shape and gq.shape == q.shape and gk.shape == k.shape and gv.shape == v.shape
        for t in (out, gq, gk, gv):
            assert not bool(t.any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_key(dtype, dev):
    """Its weight is 1 whatever the scores: the values' gradient is the sum of the rows', the others are 0 and nothing near it."""
    for Lk, lengths, mask in ((1, None, None), (50, torch.tensor([1, 1]), None), (300, torch.tensor([1, 1]), None), (64, None, torch.arange(64).expand(2, 64) == torch.tensor([[63], [5]]))):
        q, k, v, g = make(2, 70, Lk, 4, 2, 40, dtype, 37)
        out, gq, gk, gv = run(dev, q, k, v, g, lengths, mask)
        which = (0, 0) if mask is None else (63, 5)
        for n in range(2):
            assert torch.equal(out[n].cpu(), v[n, which[n]].repeat_interleave(2, 0).expand(70, 4, 40))
        assert not bool(gq.any()) and not bool(gk.any())
        want, bounds = reference(q, k, v, g, lengths, mask, 1.0 / math.sqrt(40))
        check((out, gq, gk, gv), want, bounds, str(Lk))


def test_only_some_gradients(dev):
    q, k, v, g = (t.to(dev) for t in make(1, 40, 90, 2, 2, 64, torch.bfloat16, 41))
    full = run(dev, q, k, v, g, None, None)[1:]
    for wanted in ((0,), (1,), (2,), (0, 2), (1, 2)):
        args = [t.detach().clone().requires_grad_(i in wanted) for i, t in enumerate((q, k, v))]
        grads = torch.autograd.grad(d2c.cross_attention(*args), [args[i] for i in wanted], g)
        for i, a in zip(wanted, grads):
            if 0 in wanted or i == 2:
                assert torch.equal(a, full[i]), wanted
            else:       # (delta is added up in another order where the queries' gradient is not wanted)
                assert_close(a, full[i], 2.0 ** -7, 2.0 ** -8 * full[i].float().abs().max().item(), f"{wanted} {i}")


@pytest.mark.parametrize("Lq,Lk,D", [(1, 50, 32), (37, 90, 64), (20, 40, 96)])
def test_gradients_against_differences(Lq, Lk, D, dev):
    """Along random directions of length 1 per element, float32: the loss's own error is about 1e-6 of its terms, a step of 2^-6 leaves about h^2 of
    the slope's scale."""
    q, k, v, g = (t.to(dev) for t in make(2, Lq, Lk, 2, 1, D, torch.float32, 51))
    _, mask = make_masks("mask", 1, Lk, 51)
    mask = mask.expand(2, Lk).contiguous().to(dev)
    ts = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(d2c.cross_attention(*ts, key_mask=mask), ts, g)
    h = 2.0 ** -6
    gen = torch.Generator(device=dev).manual_seed(3)
    for i in range(3):
        step = torch.randn(ts[i].shape, generator=gen, device=dev)

        def loss(sign):
            args = [t.detach() + (sign * h * step if j == i else 0) for j, t in enumerate(ts)]
            return (d2c.cross_attention(*args, key_mask=mask).double() * g.double()).sum()
        slope = ((loss(1) - loss(-1)) / (2 * h)).item()
        exact = (grads[i].double() * step.double()).sum().item()
        size = (grads[i].double() * step.double()).norm().item()
        assert abs(slope - exact) <= 5e-3 * max(size, abs(exact)), (i, slope, exact, size)


def test_float16(dev):
    q, k, v, g = make(2, 10, 30, 2, 1, 64, torch.float16, 61)
    want, bounds = reference(q.float(), k.float(), v.float(), g.float(), None, None, 1.0 / 8)
    got = run(dev, q, k, v, g, None, None)
    assert all(t.dtype == torch.float16 for t in got)
    check(got, want, [b + 2.0 ** -11 * w.abs() + 2.0 ** -24 for b, w in zip(bounds, want)])


def test_offsets_beyond_32_bits(dev):
    """Samples and positions of a memory whose elements lie more than 2^31 apart."""
    D, Lk, far = 64, 70, (1 << 31) + 64
    q, k, v, g = make(2, 40, Lk, 1, 1, D, torch.bfloat16, 71)
    want, bounds = reference(q, k, v, g, None, None, 1.0 / 8)
    row = far // (Lk - 1) // 64 * 64 + 64       # positions: the last one starts beyond 2^31 elements
    size = max(far + Lk * D, row * Lk)
    buf = torch.empty(size, dtype=torch.bfloat16, device=dev)
    for name, strides in (("samples", (far, D, D, 1)), ("positions", (0, row, D, 1))):
        def place(t):
            return torch.as_strided(buf, t.shape if name == "samples" else (1, *t.shape[1:]), strides)
        n = 2 if name == "samples" else 1
        kd = place(k[:n])
        kd.copy_(k[:n].to(dev))
        out = d2c.cross_attention(q[:n].to(dev), kd, v[:n].to(dev))
        check((out,), (want[0][:n],), (bounds[0][:n],), name + " of the keys")
        vd = place(v[:n])
        vd.copy_(v[:n].to(dev))
        out = d2c.cross_attention(q[:n].to(dev), k[:n].to(dev), vd)
        check((out,), (want[0][:n],), (bounds[0][:n],), name + " of the values")


def test_another_stream_and_graph(dev):
    q, k, v, g = (t.to(dev) for t in make(1, 1, 3000, 4, 1, 64, torch.bfloat16, 81))
    with torch.no_grad():
        here = d2c.cross_attention(q, k, v)
        s = torch.cuda.Stream(dev)
        s.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(s):
            there = d2c.cross_attention(q, k, v)
        torch.cuda.current_stream(dev).wait_stream(s)
        assert torch.equal(here, there)
        graph = torch.cuda.CUDAGraph()
        q2 = q.clone()
        with torch.cuda.graph(graph):
            out = d2c.cross_attention(q2, k, v)
        for i in range(4):
            q2.copy_(q * (1 + i))
            graph.replay()
            torch.cuda.synchronize(dev)
            assert torch.equal(out, d2c.cross_attention(q * (1 + i), k, v)), i


def test_refusals(dev):
    q, k, v, _ = (t.to(dev) for t in make(2, 4, 6, 4, 2, 32, torch.float32, 1))
    f = d2c.cross_attention
    for args, kw, text in (
            ((q[0], k, v), {}, "query must be"), ((q, k[:, :5], v), {}, "differ in shape"), ((q, k[:1], v[:1]), {}, "does not fit"),
            ((q[:, :, :3], k, v), {}, "multiple"), ((q, k.bfloat16(), v), {}, "one dtype"),
            ((q.double(), k.double(), v.double()), {}, "unsupported dtype"),
            ((q, k, v), dict(scale=0.0), "scale"), ((q, k, v), dict(scale=math.nan), "scale"),
            ((q, k, v), dict(key_lengths=torch.ones(3, dtype=torch.int32, device=dev)), "key_lengths"),
            ((q, k, v), dict(key_lengths=torch.ones(2, device=dev)), "key_lengths"),
            ((q, k, v), dict(key_mask=torch.ones(2, 6, device=dev)), "key_mask"),
            ((q, k, v), dict(key_mask=torch.ones(2, 5, dtype=torch.bool, device=dev)), "key_mask"),
            ((q.cpu(), k, v), {}, "on the GPU"), ((q, k, v), dict(key_mask=torch.ones(2, 6, dtype=torch.bool)), "on the GPU")):
        with pytest.raises(RuntimeError, match=text):
            f(*args, **kw)
    w = torch.zeros(1, 2, 1, 129, device=dev)
    with pytest.raises(RuntimeError, match="up to 128"):
        f(w, w, w)
    x = q.clone().requires_grad_()
    (gx,) = torch.autograd.grad(f(x, k, v).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
        gx.sum().backward()
