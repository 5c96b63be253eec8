"""packed_attention against the definition in float64, forward and all gradients, element by element (bounds: _packed.py)."""
import math

import pytest
import torch

import _packed
import d2conv3d_amd as d2c
from _packed import check, make, reference

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]


def run(dev, q, k, v, g, starts, key_starts=None, causal=True, frame=1, scale=None):
    args = [t.to(dev).requires_grad_() for t in (q, k, v)]
    out = d2c.packed_attention(*args, starts.to(dev), None if key_starts is None else key_starts.to(dev), causal, frame, scale)
    grads = torch.autograd.grad(out, args, g.to(dev))
    torch.cuda.synchronize(dev)
    return (out, *grads)


CASES = [
    # queries, keys (None: the same), query heads, key heads, channels, causal, frame, tokens before, behind
    ([1], None, 1, 1, 64, True, 1, 0, 0),
    ([2], None, 2, 1, 32, True, 1, 0, 0),
    ([64], None, 1, 1, 64, True, 1, 0, 0),
    ([65, 63, 1, 0, 2], None, 4, 2, 40, True, 1, 0, 0),
    ([0, 0], None, 2, 2, 24, True, 1, 3, 2),
    ([128, 129, 127], None, 1, 1, 96, True, 1, 5, 9),
    ([33, 200], None, 6, 2, 24, True, 7, 0, 0),
    ([50, 21], [200, 21], 4, 4, 72, True, 1, 0, 0),
    ([7, 1, 90], [300, 77, 100], 8, 1, 80, True, 16, 1, 0),
    ([30, 5], [10, 5], 2, 2, 64, True, 1, 0, 0),             # queries in front of their keys: rows without keys
    ([30, 5, 4], [10, 0, 7], 4, 2, 64, True, 4, 0, 0),
    ([0, 3], [40, 9], 2, 1, 128, True, 1, 0, 0),             # keys without queries
    ([70, 20], [130, 40], 3, 1, 104, False, 1, 0, 3),
    ([9], [31], 2, 2, 1, False, 1, 0, 0),
    ([20, 60], None, 3, 1, 7, True, 5, 2, 2),
    ([65], None, 2, 2, 33, True, 64, 0, 0),
    ([100], None, 2, 1, 100, True, 1000, 0, 0),              # one frame longer than the sequence
    ([31, 140], None, 1, 1, 127, True, 1, 0, 0),
    ([1500], None, 2, 1, 64, True, 1, 0, 0),                 # walks that are shared
    ([40, 300], [3000, 2000], 1, 1, 64, True, 1, 0, 0),
    ([700], None, 2, 2, 128, True, 100, 0, 0),
    ([2000], [2000], 1, 1, 40, False, 1, 0, 0),
    ([300], None, 12, 3, 32, True, 1, 0, 0),
    ([60], None, 5, 1, 88, True, 1, 0, 0),
    ([11, 3], None, 160, 1, 16, True, 1, 0, 0),              # more rows to a token than a tile has
    ([1] * 70 + [3, 0, 130], None, 2, 1, 48, True, 1, 1, 1),
    ([2, 3, 1, 0] * 60, None, 1, 1, 8, True, 2, 0, 0),
    ([526], [984], 8, 8, 120, True, 1, 0, 0),
    ([1, 2, 0, 3] * 1100, None, 1, 1, 8, True, 1, 2, 1),     # more sequences than two steps of the search tell apart
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{c[2]}-{c[3]}-{c[4]}-{c[5]}-{c[6]}")
def test_forward_and_gradients(case, dtype, dev):
    print("packed_attention", case, dtype, flush=True)
    lq, lk, hq, hkv, D, causal, frame, before, behind = case
    q, k, v, g, starts, key_starts = make(lq, lq if lk is None else lk, hq, hkv, D, dtype, sum(lq) + D, before, behind)
    want, bounds = reference(q, k, v, g, starts, key_starts, causal, frame)
    other = None if lk is None else key_starts
    got = run(dev, q, k, v, g, starts, other, causal, frame)
    check(got, want, bounds, str(case))
    again = run(dev, q, k, v, g, starts.long(), other, causal, frame)      # (and whole numbers of 64 bits)
    for a, b in zip(got, again):
        assert torch.equal(a, b)             # sums in one order
    with torch.no_grad():
        alone = d2c.packed_attention(*(t.to(dev) for t in (q, k, v)), starts.to(dev), None if other is None else other.to(dev), causal, frame)
    assert torch.equal(alone, got[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size,scale", [(12.0, None), (1.0, 3.0), (1.0, 1e-3)])
def test_scores_of_any_size(size, scale, dtype, dev):
    q, k, v, g, starts, _ = make([37, 150], [37, 150], 2, 1, 64, dtype, 5)
    q = (q.float() * size).to(dtype)
    want, bounds = reference(q, k, v, g, starts, starts, scale=scale)
    check(run(dev, q, k, v, g, starts, scale=scale), want, bounds, f"{size} {scale}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 40, 64, 72, 104, 128])
@pytest.mark.parametrize("garbage", [math.nan, math.inf, -math.inf, "lowest"])
def test_what_is_not_read_has_no_influence(garbage, D, dtype, dev):
    """A token's key, value, query and gradient of the output that are no numbers: what does not read it, and what it does not read, as without it."""
    lq, lk = [150, 40, 70], [150, 90, 70]
    q, k, v, g, starts, key_starts = make(lq, lk, 4, 2, D, dtype, 9)
    want, bounds = reference(q, k, v, g, starts, key_starts, frame=3)
    value = torch.finfo(dtype).min if garbage == "lowest" else garbage
    tokens = [(0, 100), (1, 70)]             # sequence, token
    fine = [torch.ones(t.shape[0], dtype=torch.bool) for t in (q, q, k, v)]
    dirty = [t.clone() for t in (q, k, v, g)]
    for s, token in tokens:
        row, key = int(starts[s]) + token - (lk[s] - lq[s]), int(key_starts[s]) + token
        dirty[0][row], dirty[1][key], dirty[2][key], dirty[3][row] = (value,) * 4
        first = token // 3 * 3               # the first token that reads it, and the last that it reads
        for i in (0, 1):
            fine[i][int(starts[s]) + first - (lk[s] - lq[s]):int(starts[s + 1])] = False
        for i in (2, 3):                     # keys that rows read whose gradients are none
            fine[i][int(key_starts[s]):int(key_starts[s + 1])] = False
    got = run(dev, *dirty, starts, key_starts, frame=3)
    check(got, want, bounds, f"{garbage}", fine)
    # the values' gradients where the weights are numbers: a gradient of the output alone that is none
    dirty = [q, k, v, g.clone()]
    fine = [torch.ones(t.shape[0], dtype=torch.bool) for t in (q, q, k, v)]
    for s, token in tokens:
        row = int(starts[s]) + token - (lk[s] - lq[s])
        dirty[3][row] = value
        fine[1][row] = False
        for i in (2, 3):
            fine[i][int(key_starts[s]):int(key_starts[s]) + token // 3 * 3 + 3] = False
    got = run(dev, *dirty, starts, key_starts, frame=3)
    check(got, want, bounds, f"gradient {garbage}", fine)
    # ... and a query alone
    dirty = [q.clone(), k, v, g]
    for s, token in tokens:
        dirty[0][int(starts[s]) + token - (lk[s] - lq[s])] = value
        fine[0][int(starts[s]) + token - (lk[s] - lq[s])] = False
    got = run(dev, *dirty, starts, key_starts, frame=3)
    check(got, want, bounds, f"query {garbage}", fine)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_infinities_that_are_read(D, dtype, dev):
    """An infinite value makes its channel infinite for those that read it, and no other; a key whose score is -infinity has a weight of 0; an infinite gradient
    of the output makes its channel of the values' gradient infinite."""
    q, k, v, g, starts, _ = make([200, 30], [200, 30], 2, 2, D, dtype, 11)
    v[100, 0, 5], v[150, 0, 6] = math.inf, -math.inf
    want, bounds = reference(q, k, torch.where(v.isinf(), 0, v), g, starts, starts)
    out = run(dev, q, k, v, g, starts)[0].double().cpu()
    assert bool((out[100:200, 0, 5] == math.inf).all()) and bool((out[150:200, 0, 6] == -math.inf).all())
    # (its weight is not among the others: compare rows that do not read it, and other channels with the value as it is)
    free = torch.ones_like(out, dtype=torch.bool)
    free[100:200, 0, 5] = free[150:200, 0, 6] = False
    assert bool(((out - want[0]).abs() <= 1.05 * bounds[0] + 1e-30)[free].all())
    # a key of -infinity against positive queries
    q, k, v, g, starts, _ = make([200, 30], [200, 30], 2, 2, D, dtype, 12)
    q[:, :, 3] = q[:, :, 3].abs() + 0.1
    k[100, 0, 3] = -math.inf
    other = k.clone()
    other[100, 0] = 0
    other[100, 0, 3] = -1e4                  # a score so low that its weight is 0 in any type
    want, bounds = reference(q, other, v, g, starts, starts)
    got = run(dev, q, k, v, g, starts)
    assert bool(((got[0].double().cpu() - want[0]).abs() <= 1.05 * bounds[0] + 1e-30)[torch.arange(230) != 100].all())
    assert not bool(got[0].isnan().any())
    # its row of the queries' gradient: 0 times infinity in that channel, for those that read it
    nan = got[1].isnan().cpu()
    assert bool(nan[100:200, 0, 3].all()) and int(nan.sum()) == 100
    # an infinite gradient of the output
    q, k, v, g, starts, _ = make([200, 30], [200, 30], 2, 2, D, dtype, 13)
    g[120, 1, 7] = math.inf
    gv = run(dev, q, k, v, g, starts)[3].cpu()
    assert bool((gv[:121, 1, 7] == math.inf).all())
    free = torch.ones_like(gv, dtype=torch.bool)
    free[:121, 1, 7] = False
    assert bool(gv[free].isfinite().all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_of_one_key_have_exact_zeros(dtype, dev):
    q, k, v, g, starts, key_starts = make([1, 5, 1, 3], [1, 1, 1, 3], 4, 2, 64, dtype, 14)
    out, gq, gk, gv = run(dev, q, k, v, g, starts, key_starts)
    for row, key in ((0, 0), (5, 1), (6, 2), (7, 3)):
        assert torch.equal(out[row].cpu(), v[key].repeat_interleave(2, 0)) and not bool(gq[row].any())
    assert not bool(out[1:5].any()) and not bool(gq[1:5].any()) and not bool(gk[:3].any()) and bool(gk[3:].any())


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype, dev):
    """Heads that are parts of one projection, at odd places, tokens that go backwards in memory for all that matters, a repeated key head."""
    D, hq, hkv = 40, 4, 2
    q, k, v, g, starts, _ = make([70, 33], [70, 33], hq, hkv, D, dtype, 21)
    want = run(dev, q, k, v, g, starts)
    wide = torch.full((103, 2, hq + 2 * hkv, D + 1), math.nan, dtype=dtype, device=dev)
    for t, a, b in ((q, 0, hq), (k, hq, hq + hkv), (v, hq + hkv, hq + 2 * hkv)):
        wide[:, 1, a:b, 1:] = t.to(dev)
    wide.requires_grad_()
    parts = [wide[:, 1, a:b, 1:] for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv))]
    out = d2c.packed_attention(*parts, starts.to(dev))
    grad, = torch.autograd.grad(out, wide, g.to(dev))
    assert torch.equal(out, want[0])
    for x, (a, b) in zip(want[1:], ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv))):
        assert torch.equal(grad[:, 1, a:b, 1:], x)
    # channels that are not adjacent are copied; a gradient that is broadcast
    apart = [t.to(dev).transpose(1, 2).contiguous().transpose(1, 2).requires_grad_() for t in (q, k, v)]
    out = d2c.packed_attention(*apart, starts.to(dev))
    assert torch.equal(out, want[0])
    out.sum().backward()
    ones = run(dev, q, k, v, torch.ones_like(g), starts)
    for a, b in zip(apart, ones[1:]):
        assert torch.equal(a.grad, b)
    # one key and value for all tokens
    one = [t[:1].to(dev).requires_grad_() for t in (k, v)]
    got = torch.autograd.grad(d2c.packed_attention(q.to(dev), *(t.expand(103, -1, -1) for t in one), starts.to(dev)), one, g.to(dev))
    exact, bounds = reference(q, k[:1].expand(103, -1, -1), v[:1].expand(103, -1, -1), g, starts, starts)
    for a, e, b in zip(got, exact[2:], bounds[2:]):
        # (each token's gradient is within its bound -- without the queries' gradient delta is summed in another order, so that no bits can be compared -- and
        # autograd adds them up: 103 float32 additions, and one rounding to the type)
        b = b.sum(0, keepdim=True) + 103 * 2.0 ** -24 * (e.abs() + b).sum(0, keepdim=True)
        a = a.double().cpu()
        assert bool(((a - e.sum(0, keepdim=True)).abs() <= b + torch.finfo(dtype).eps / 2 * a.abs()).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_far_apart(dtype, dev):
    """Tokens whose elements lie beyond offsets of 32 bits inside a tile, and sequences that do from the first."""
    D, tokens = 64, 40
    q, k, v, g, starts, _ = make([25, 15], [25, 15], 2, 1, D, dtype, 22)
    exact = reference(q, k, v, g, starts, starts)
    step = 2 ** 26 if dtype == torch.bfloat16 else 2 ** 25
    pool = torch.empty(step * tokens + 1024, dtype=dtype, device=dev)
    far = [pool[at:].as_strided(t.shape, (step, D, 1)) for t, at in ((q, 0), (k, 256), (v, 512))]
    with torch.no_grad():
        for a, b in zip(far, (q, k, v)):
            a.copy_(b)
    with torch.no_grad():
        check([d2c.packed_attention(*far, starts.to(dev))], *(x[:1] for x in exact))
    step = 2 ** 16
    tokens = 2 ** 31 // step + 2 ** 13
    del pool, far
    pool = torch.empty(step * tokens, dtype=dtype, device=dev)
    far = [pool[at:].as_strided((tokens, *t.shape[1:]), (step, D, 1)) for t, at in ((q, 0), (k, 256), (v, 512))]
    with torch.no_grad():
        for a, b in zip(far, (q, k, v)):
            a[-40:].copy_(b)
    grad = torch.zeros(tokens, 2, D, dtype=dtype, device=dev)
    grad[-40:] = g.to(dev)
    far = [t.detach().requires_grad_() for t in far]
    out = d2c.packed_attention(*far, (starts + tokens - 40).to(dev))
    got = torch.autograd.grad(out, far, grad)
    check([t[-40:] for t in (out, *got)], *exact)
    assert not any(bool(t[:-40].any()) for t in (out, *got))


def test_differences(dev):
    """Gradients against central differences of the forward pass, float32 sums in 64 bits."""
    q, k, v, g, starts, key_starts = make([40, 9], [60, 9], 4, 2, 32, torch.float32, 23)
    _, *grads = run(dev, q, k, v, g, starts, key_starts, frame=5)
    gen = torch.Generator().manual_seed(24)
    for i, (t, grad) in enumerate(zip((q, k, v), grads)):
        u, slope = torch.randn(t.shape, generator=gen), grad.cpu()
        u = u / u.norm() + slope / slope.norm()
        sides = []
        for sign in (1, -1):
            moved = [x if j != i else x + sign * 0.02 * u for j, x in enumerate((q, k, v))]
            with torch.no_grad():
                out = d2c.packed_attention(*(x.to(dev) for x in moved), starts.to(dev), key_starts.to(dev), frame=5)
            sides.append((out.double().cpu() * g.double()).sum())
        want = (slope.double() * u.double()).sum().item()
        # (6272 outputs, each off by 1e-5 at most, times a gradient of about 1, over 0.04: 1.6 if all were off the same way; slopes are 30 and more.  Curvature: 0.02^2.)
        assert abs(((sides[0] - sides[1]) / 0.04).item() - want) < 0.03 * want, (i, want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_some_gradients_only(dtype, dev):
    q, k, v, g, starts, _ = make([70, 200, 1], [70, 200, 1], 4, 2, 72, dtype, 25)
    want = run(dev, q, k, v, g, starts)
    for wanted in ((0,), (1,), (2,), (0, 2), (1, 2)):
        args = [t.to(dev).requires_grad_(i in wanted) for i, t in enumerate((q, k, v))]
        grads = torch.autograd.grad(d2c.packed_attention(*args, starts.to(dev)), [args[i] for i in wanted], g.to(dev))
        for i, a in zip(wanted, grads):
            # (delta alone is summed in another order where the queries' gradient is not wanted)
            if 0 in wanted or i == 2:
                assert torch.equal(a, want[1 + i]), wanted
            else:
                check([a], *([x[1 + i]] for x in reference(q, k, v, g, starts, starts)), str(wanted))


@pytest.mark.parametrize("dtype", DTYPES)
def test_captured_and_replayed(dtype, dev):
    """A training step's share in a graph, with other numbers and other starts in the same tensors on each replay."""
    q, k, v, g, starts, _ = make([300, 20, 180], [300, 20, 180], 4, 2, 64, dtype, 26)
    static = [t.to(dev) for t in (q, k, v, g, starts)]
    leaves = [t.requires_grad_() for t in static[:3]]

    def step():
        out = d2c.packed_attention(*leaves, static[4], frame=10)
        return (out, *torch.autograd.grad(out, leaves, static[3]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed, lengths in ((27, [300, 20, 180]), (28, [1, 499, 0]), (29, [100, 100, 300])):
        q, k, v, g, starts, _ = make(lengths, lengths, 4, 2, 64, dtype, seed)
        with torch.no_grad():
            for a, b in zip(static, (q, k, v, g, starts)):
                a.copy_(b)
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(captured, run(dev, q, k, v, g, starts, frame=10)):
                assert torch.equal(a, b), lengths


def test_starts_that_do_not_rise(dev):
    """Results of no meaning, from inside the tensors: starts of any numbers run, and calls behind them are what they are."""
    q, k, v, g, starts, _ = make([100, 100], [100, 100], 2, 1, 64, torch.float32, 30)
    for bad in ([0, 150, 100], [200, 100, 0], [-50, 1000, 20], [2 ** 31 - 1, -2 ** 31, 5]):
        for a, b in ((bad, bad), ([0, 100, 200], bad), (bad, [0, 100, 200])):
            run(dev, q, k, v, g, torch.tensor(a, dtype=torch.int32), torch.tensor(b, dtype=torch.int32))
    check(run(dev, q, k, v, g, torch.tensor([-7, 100, 300], dtype=torch.int32)), *reference(q, k, v, g, starts, starts))


def test_both_routes(dev, monkeypatch):
    from d2conv3d_amd import _ops
    q, k, v, g, starts, key_starts = make([50, 7], [60, 7], 4, 2, 40, torch.bfloat16, 31)
    want = run(dev, q, k, v, g, starts, key_starts, frame=2)
    monkeypatch.setattr(_ops, "_native", type("None_", (), {"__getattr__": lambda self, name: lambda *a: None})())
    for a, b in zip(want, run(dev, q, k, v, g, starts, key_starts, frame=2)):
        assert torch.equal(a, b)


def test_float16(dev):
    q, k, v, g, starts, _ = make([50, 7], [50, 7], 4, 2, 40, torch.float16, 32)
    got = run(dev, q, k, v, g, starts)
    wide = run(dev, q.float(), k.float(), v.float(), g.float(), starts)
    for a, b in zip(got, wide):
        assert a.dtype == torch.float16 and torch.equal(a, b.half())


def test_no_tokens(dev):
    for T, Tk in ((0, 0), (0, 5), (5, 0)):
        q, k = torch.zeros(T, 2, 16, device=dev, requires_grad=True), torch.zeros(Tk, 1, 16, device=dev, requires_grad=True)
        starts, key_starts = (torch.tensor([0, n], device=dev) for n in (T, Tk))
        out = d2c.packed_attention(q, k, k * 2, starts, key_starts)
        gq, gk = torch.autograd.grad(out, (q, k), torch.ones_like(out))
        assert out.shape == q.shape and not bool(out.any()) and not bool(gq.any()) and gk.shape == k.shape and not bool(gk.any())
    # no sequence at all
    q = torch.ones(4, 2, 16, device=dev)
    assert not bool(d2c.packed_attention(q, q, q, torch.tensor([0], device=dev)).any())


def test_what_is_kept_may_not_change(dev):
    q, k, v, g, starts, _ = make([20], [20], 2, 1, 16, torch.float32, 33)
    for changed in range(4):
        args = [t.to(dev) for t in (q, k, v)]
        leaf = args[0].clone().requires_grad_()
        first = starts.to(dev)
        out = d2c.packed_attention(leaf * 1.0, *args[1:], first)
        (args[1], args[2], first, out.detach())[changed].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.backward(g.to(dev))
