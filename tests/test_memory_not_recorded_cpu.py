"""The memory's functions refuse what they would be silently left out of: torch.jit.trace and forward-mode differentiation.  Without a GPU."""
import pytest
import torch
from torch.autograd import forward_ad

import d2conv3d_amd as d2c


class OnTheGpu(torch.Tensor):
    """A CPU tensor that says it is on the GPU: what the argument checks look at, with no memory touched."""
    is_cuda = True


def memory():
    m = d2c.PagedMemory.empty(2, 40, 2, 16, page=8, dtype=torch.float32, device="cpu")
    for name in d2c.PagedMemory.__slots__:
        setattr(m, name, getattr(m, name).as_subclass(OnTheGpu))
    return m


CALLS = {
    "memory_attention": lambda m, t: d2c.memory_attention(t, m),
    "tracked memory_attention": lambda m, t: d2c.memory_attention(t, m, track=True),
    "memory_append": lambda m, t: d2c.memory_append(m, t, t) or t,
    "packed memory_append": lambda m, t: d2c.memory_append(m, t, t, torch.tensor([0, 1, 2])) or t,
    "memory_evict": lambda m, t: d2c.memory_evict(m, 3) or t,
}


@pytest.mark.parametrize("call", CALLS)
def test_traced(call):
    m = memory()
    with pytest.raises(RuntimeError, match="is not recorded by torch.jit.trace"):
        torch.jit.trace(lambda t: CALLS[call](m, t) * 1.0, (torch.ones(2, 2, 16),), check_trace=False)


@pytest.mark.parametrize("call", [c for c in CALLS if c != "memory_evict"])
def test_tangent_of_a_token(call):
    with forward_ad.dual_level():
        t = forward_ad.make_dual(torch.ones(2, 2, 16), torch.ones(2, 2, 16))
        with pytest.raises(RuntimeError, match="no forward-mode tangent"):
            CALLS[call](memory(), t)


@pytest.mark.parametrize("field", ["key", "value", "usage"])
@pytest.mark.parametrize("call", CALLS)
def test_tangent_of_the_memory(call, field):
    with forward_ad.dual_level():
        m = memory()
        plain = torch.zeros(getattr(m, field).shape)
        setattr(m, field, forward_ad.make_dual(plain, torch.ones_like(plain)))
        with pytest.raises(RuntimeError, match="no forward-mode tangent"):
            CALLS[call](m, torch.ones(2, 2, 16))
