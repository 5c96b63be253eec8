"""Evictions of long streams whose slots share the border's usage, or its leading bits: a memory that was read without `track` has a usage of 0 everywhere.  More slots than the
kernel's list of candidates holds, and than it takes at a time; the border among the ties, before them and behind them."""
import pytest
import torch

import _memory
from _memory import assert_same, make, on

pytestmark = pytest.mark.gpu


def usage_of(kind, shape, gen):
    if kind == "zeros":
        return torch.zeros(shape)
    if kind == "few":
        return torch.randint(0, 3, shape, generator=gen) / 4.0
    if kind == "most equal":      # (a few above and below what the others have)
        x = torch.rand(shape, generator=gen)
        return torch.where(x < 0.03, 2.0, torch.where(x > 0.95, 1e-3, 0.25))
    # numbers that agree in their leading 11 bits, and some more
    return 1.0 + torch.randint(0, {"near": 1 << 12, "nearer": 1 << 9}[kind], shape, generator=gen) * 2.0 ** -23


@pytest.mark.parametrize("usage", ["zeros", "few", "most equal", "near", "nearer"])
@pytest.mark.parametrize("length,page,keeps", [(6145, 16, (6144, 1)), (7001, 64, (3000, 6990)), (20000, 50, (10007,)), (66000, 64, (65537, 300)), (70001, 16, (35000,))])
def test_ties(usage, length, page, keeps, dev):
    for keep in keeps:
        for recent in (0, keep // 3):
            m = make([length], page, 1, 4, torch.float32, seed=length + keep)
            m["usage"] = usage_of(usage, m["usage"].shape, torch.Generator().manual_seed(keep))
            memory = on(dev, m)
            print("memory_evict", usage, length, page, keep, recent, flush=True)
            memory.evict(keep, recent)
            assert_same(memory, _memory.evict(m, keep, recent), f"{keep} {recent}")


def test_never_tracked(dev):
    """Streams of several heads that were read without `track`: the newest stay, and of the others those in the lowest slots."""
    m = make([9000, 6500, 100], 64, 3, 16, torch.bfloat16, seed=4)
    m["usage"] = torch.zeros_like(m["usage"])
    memory = on(dev, m)
    memory.attend(torch.randn(3, 6, 16, generator=torch.Generator().manual_seed(5)).bfloat16().to(dev))
    assert not bool(memory.usage.any())
    memory.evict(6000, 1000)
    assert_same(memory, _memory.evict(m, 6000, 1000))
