"""layer_norm, rotary3d and cross_attention through the native binding and through the Python functions: the same kernels on the
same tensors, so the same bits; on a stream of their own, with what is kept for the backward pass moved to host memory, and with
gradients that are views."""
import contextlib

import pytest
import torch

import d2conv3d_amd as d2c
from d2conv3d_amd import attention

pytestmark = pytest.mark.gpu


def _rn(seed, *shapes, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(*s, generator=gen).to(dtype) for s in shapes]


def _norm(dtype):
    return d2c.layer_norm, lambda seed: _rn(seed, (3, 41, 72), (72,), (72,), dtype=dtype)


def _rotary(dtype):
    return lambda x: d2c.rotary3d(x, (2, 3, 7), interleaved=True), lambda seed: _rn(seed, (2, 42, 3, 40), dtype=dtype)


def _attention(dtype, Lq=90):
    lengths, mask = torch.tensor([200, 77]), torch.arange(200).expand(2, 200) % 3 != 1
    return (lambda q, k, v: d2c.cross_attention(q, k, v, lengths.to(q.device), mask.to(q.device)),
            lambda seed: _rn(seed, (2, Lq, 6, 40), (2, 200, 3, 40), (2, 200, 3, 40), dtype=dtype))


ENTRIES = {f"{name}_{str(dtype)[6:]}": make(dtype) for dtype in (torch.float32, torch.bfloat16)
           for name, make in (("norm", _norm), ("rotary", _rotary), ("attention", _attention), ("token", lambda t: _attention(t, 1)))}


@contextlib.contextmanager
def python_route():
    with pytest.MonkeyPatch.context() as mp:
        mp.setattr(attention, "_try_native", lambda *a: None)
        yield


def _step(fn, ts, grad=None):
    out = fn(*ts)
    if grad is None:
        (grad,) = _rn(9, out.shape)
    out.backward(grad.to(out))
    return [out.detach()] + [t.grad for t in ts]


def _side_stream(fn, ts):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _step(fn, ts)
    torch.cuda.current_stream().wait_stream(side)
    return got


def _offloaded(fn, ts):
    dev = ts[0].device
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().cpu(), lambda t: t.to(dev)):
        out = fn(*ts)
    (grad,) = _rn(9, out.shape)
    out.backward(grad.to(out))
    return [out.detach()] + [t.grad for t in ts]


def _checkpointed(fn, ts):
    from torch.utils.checkpoint import checkpoint
    return _step(lambda *a: checkpoint(fn, *a, use_reentrant=False), ts)


def _strided_gradient(fn, ts):
    """The same gradient, as every second of the elements of a wider one."""
    out = fn(*ts)
    (grad,) = _rn(9, out.shape)
    wide = torch.full((*out.shape, 2), float("nan"), device=out.device, dtype=out.dtype)
    wide[..., 0] = grad.to(out)
    out.backward(wide[..., 0])
    return [out.detach()] + [t.grad for t in ts]


@pytest.mark.parametrize("way", [_step, _side_stream, _offloaded, _checkpointed, _strided_gradient])
@pytest.mark.parametrize("entry", ENTRIES)
def test_both_routes_give_the_same_bits(entry, way, dev):
    fn, tensors = ENTRIES[entry]

    def leaves():
        return [t.to(dev).requires_grad_() for t in tensors(3)]
    with python_route():
        want = _step(fn, leaves())
        python = way(fn, leaves())
    native = way(fn, leaves())
    for w, p, n in zip(want, python, native):
        assert torch.equal(w, p) and torch.equal(w, n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_kept_tensors_that_come_back_with_other_strides(dtype, dev):
    """Inputs that are views at wide strides or broadcast, kept in host memory (which makes them dense): the same gradients."""
    def dense(t):
        return t.detach().cpu().contiguous()

    def spread(t):      # the same values, channels adjacent, everything else far apart
        wide = torch.full((*t.shape[:-2], t.size(-2) + 1, t.size(-1) + 8), float("nan"), device=dev, dtype=dtype)
        wide[..., :-1, :-8] = t.to(dev)
        return wide[..., :-1, :-8]

    def step(fn, ts, hooks):
        ts = [t.detach().requires_grad_() for t in ts]
        with torch.autograd.graph.saved_tensors_hooks(dense, lambda t: t.to(dev)) if hooks else contextlib.nullcontext():
            out = fn(*ts)
        (grad,) = _rn(9, out.shape)
        out.backward(grad.to(out))
        return [t.grad for t in ts]
    rows, w, b = _rn(3, (41, 72), (72,), (72,), dtype=dtype)
    q, k, v = _rn(4, (2, 90, 6, 40), (2, 200, 3, 40), (2, 200, 3, 40), dtype=dtype)
    for fn, ts in ((d2c.layer_norm, (spread(rows), w.to(dev), b.to(dev))), (d2c.layer_norm, (rows[:1].to(dev).expand(5, 72), w.to(dev), b.to(dev))),
                   (d2c.cross_attention, (spread(q), spread(k), spread(v))),
                   (d2c.cross_attention, (q[:, :1].to(dev).expand(2, 90, 6, 40), k[:1].to(dev).expand(2, 200, 3, 40), spread(v)))):
        for route in (contextlib.nullcontext, python_route):
            with route():
                for a, c in zip(step(fn, ts, False), step(fn, ts, True)):
                    assert torch.equal(a, c)


def test_tokens_of_a_feature_map(dev):
    """Channels far apart (a map [N, C, T, H, W] as tokens): read as they are or copied, the results are the dense tensor's."""
    (x, g, w, b, turn, tg) = (t.to(dev) for t in _rn(6, (2, 72, 41), (2, 41, 72), (72,), (72,), (2, 40, 42, 3), (2, 42, 3, 40)))
    for fn, dense, grad in ((lambda t: d2c.layer_norm(t, w, b), lambda t: t.transpose(1, 2), g),
                            (lambda t: d2c.rotary3d(t, (2, 3, 7)), lambda t: t.permute(0, 2, 3, 1), tg)):
        base = x if grad is g else turn
        for route in (contextlib.nullcontext, python_route):
            with route():
                far = base.clone().requires_grad_()
                out = fn(dense(far))
                out.backward(grad)
                near = dense(base).contiguous().requires_grad_()
                want = fn(near)
                want.backward(grad)
                assert torch.equal(out, want) and torch.equal(dense(far.grad), near.grad)


@pytest.mark.parametrize("entry", ENTRIES)
def test_a_changed_input_is_noticed(entry, dev):
    fn, tensors = ENTRIES[entry]
    if entry.startswith("rotary"):
        pytest.skip("the gradient of a turn needs no input")
    for route in (contextlib.nullcontext, python_route):
        with route():
            ts = [t.to(dev).requires_grad_() for t in tensors(3)]
            out = fn(*ts)
            with torch.no_grad():
                ts[0].add_(1.0)
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                out.sum().backward()


@pytest.mark.parametrize("entry", ENTRIES)
def test_the_same_call_twice_gives_the_same_bits(entry, dev):
    fn, tensors = ENTRIES[entry]
    first, second = (_step(fn, [t.to(dev).requires_grad_() for t in tensors(5)]) for _ in range(2))
    for a, b in zip(first, second):
        assert torch.equal(a, b)
