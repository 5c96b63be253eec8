"""The memory's functions on the GPU: refused where torch.jit.trace would record them or a forward-mode tangent would be lost, and nothing is changed."""
import pytest
import torch
from torch.autograd import forward_ad

from _memory import FIELDS, assert_same, make, on

pytestmark = pytest.mark.gpu

CALLS = [lambda m, q, k: m.attend(q), lambda m, q, k: m.attend(q, track=True), lambda m, q, k: m.append(k, k) and q, lambda m, q, k: m.evict(5) and q]


@pytest.mark.parametrize("call", range(len(CALLS)))
def test_traced(call, dev):
    m = make([40, 9], 16, 2, 32, torch.float32, seed=1)
    memory = on(dev, m)
    q, k = torch.randn(2, 4, 32, device=dev), torch.randn(2, 2, 32, device=dev)
    with pytest.raises(RuntimeError, match="is not recorded by torch.jit.trace"):
        torch.jit.trace(lambda q, k: CALLS[call](memory, q, k) * 1.0, (q, k), check_trace=False)
    assert_same(memory, m)


@pytest.mark.parametrize("call,which", [(0, "query"), (1, "query"), (2, "new key"), *((call, f) for call in range(len(CALLS)) for f in ("key", "value", "usage"))])
def test_tangents(call, which, dev):
    m = make([40, 9], 16, 2, 32, torch.float32, seed=1, garbage=0.0)
    memory = on(dev, m)
    q, k = torch.randn(2, 4, 32, device=dev), torch.randn(2, 2, 32, device=dev)
    with forward_ad.dual_level():
        other = on(dev, m)
        for f in FIELDS:
            setattr(other, f, getattr(memory, f))

        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        if which in FIELDS:
            setattr(other, which, dual(getattr(memory, which)))
        with pytest.raises(RuntimeError, match="no forward-mode tangent"):
            CALLS[call](other, dual(q) if which == "query" else q, dual(k) if which == "new key" else k)
    assert_same(memory, m)
