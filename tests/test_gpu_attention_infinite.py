"""Infinite values among what cross_attention reads, where the definition has a finite result all the same.  A key with a channel of -infinity that meets
positive queries has scores of -infinity: its weight is 0, as if it were not to be read.  Outputs and gradients are those of the call without it, but for the
queries' gradient in that channel, where 0 times infinity is no number.  An infinite value makes its channel of the outputs infinite, and no
other.  Bounds: test_gpu_attention.py."""
import math

import pytest
import torch

import d2conv3d_amd as d2c
from test_gpu_attention import check, make, reference, run

pytestmark = pytest.mark.gpu


def without_weight(sizes, D, dtype, channel, masked, dev):
    N, Lq, Lk, Hq, Hkv = sizes
    q, k, v, g = make(*sizes, D, dtype, seed=sum(sizes) + D)
    q[..., channel] = q[..., channel].abs() + 0.125
    gen = torch.Generator().manual_seed(11)
    mask = torch.rand(N, Lk, generator=gen) < 0.7 if masked else torch.ones(N, Lk, dtype=torch.bool)
    gone = mask & (torch.rand(N, Lk, generator=gen) < 0.2)
    assert bool(gone.any()) and bool((mask & ~gone).any(1).all())
    want, bounds = reference(q, k, v, g, None, mask & ~gone, 1.0 / math.sqrt(D))
    k[..., channel][gone] = -math.inf
    got = run(dev, q, k, v, g, None, mask if masked else None)
    assert bool(got[1][..., channel].isnan().all())
    rest = [c for c in range(D) if c != channel]
    got, want, bounds = ([t if i != 1 else t[..., rest] for i, t in enumerate(ts)] for ts in (got, want, bounds))
    check(got, want, bounds, f"{sizes} {D} {channel} {masked}")
    for i in (2, 3):
        assert not bool(got[i].cpu()[gone].any())


# (rows of a key head: up to 8, up to 32, more; few keys; more than 2^22 scores)
SIZES = [(2, 1, 300, 2, 1), (2, 20, 300, 2, 2), (1, 200, 333, 2, 1), (2, 40, 60, 2, 1), (1, 1100, 2000, 2, 2)]


@pytest.mark.parametrize("D", [8, 24, 33, 40, 56, 64, 72, 88, 104, 120, 128])
def test_keys_at_minus_infinity_bfloat16(D, dev):
    for sizes in SIZES:
        for channel, masked in ((D - 1, False), (max(D - 6, 0), True), (0, False)):
            without_weight(sizes, D, torch.bfloat16, channel, masked, dev)


@pytest.mark.parametrize("D", [8, 24, 33, 40, 64, 72, 96, 104, 128])
def test_keys_at_minus_infinity_float32(D, dev):
    for sizes in SIZES[:4]:
        for channel, masked in ((D - 1, False), (max(D - 6, 0), True), (0, False)):
            without_weight(sizes, D, torch.float32, channel, masked, dev)


def infinite_value(sizes, D, dtype, mask, gone, dev):
    """`gone` [N, Lk]: the keys whose value is infinite in one channel, of which a sample has no two of opposite sign"""
    N, Lq, Lk, Hq, Hkv = sizes
    q, k, v, g = make(*sizes, D, dtype, seed=sum(sizes) + D)
    want, bounds = reference(q, k, v, g, None, mask, 1.0 / math.sqrt(D))
    out, bound = want[0], bounds[0]
    channel, sign = D - 3, 1 - 2 * (torch.arange(N) % 2)
    v[..., channel] = torch.where(gone[..., None], (sign * math.inf)[:, None, None].to(dtype), v[..., channel])
    with torch.no_grad():
        got = d2c.cross_attention(q.to(dev), k.to(dev), v.to(dev), key_mask=None if mask is None else mask.to(dev)).double().cpu()
    infinite = (sign * math.inf)[:, None, None].expand(N, Lq, Hq).double()
    assert torch.equal(got[..., channel], infinite), (sizes, D, got[..., channel].isnan().sum())
    rest = [c for c in range(D) if c != channel]
    check((got[..., rest],), (out[..., rest],), (bound[..., rest],), f"{sizes} {D}")


@pytest.mark.parametrize("D", [8, 24, 33, 40, 64, 96, 104, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinite_values(dtype, D, dev):
    for sizes in ((2, 1, 384, 2, 1), (2, 20, 384, 2, 2), (2, 200, 384, 2, 1), (2, 200, 64, 2, 1)):
        gone = torch.zeros(sizes[0], sizes[2], dtype=torch.bool)
        gone[:, 17], gone[1, 60] = True, True
        infinite_value(sizes, D, dtype, None, gone, dev)


@pytest.mark.parametrize("D", [8, 24, 33, 40, 64, 96, 104, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinite_values_beside_keys_that_are_not_read(dtype, D, dev):
    """... in tiles that are not whole, by their end or by the mask; every key that is read is one of those whose value is infinite in turn"""
    for sizes in ((2, 1, 333, 2, 1), (2, 20, 333, 2, 2), (2, 200, 333, 2, 1), (2, 200, 50, 2, 1), (2, 20, 50, 2, 1), (1, 1100, 2000, 2, 2)):
        N, Lk = sizes[0], sizes[2]
        mask = torch.rand(N, Lk, generator=torch.Generator().manual_seed(5)) < 0.5
        infinite_value(sizes, D, dtype, mask, mask, dev)                          # (weights above 0 all: the scores are near each other)
        gone = torch.zeros(N, Lk, dtype=torch.bool)
        gone[:, Lk - 1] = True
        infinite_value(sizes, D, dtype, None, gone, dev)


@pytest.mark.parametrize("D", [8, 33, 40, 64, 104, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinite_gradients(dtype, D, dev):
    """grad_out of the last row infinite in a channel: that channel of the values' gradients is infinite, the others are as they were."""
    for sizes in ((2, 3, 333, 2, 1), (1, 70, 300, 3, 1), (2, 20, 50, 2, 2), (1, 1111, 2000, 2, 2)):
        q, k, v, g = make(*sizes, D, dtype, seed=sum(sizes) + D)
        want, bounds = reference(q, k, v, g, None, None, 1.0 / math.sqrt(D))
        g[:, -1, :, D - 2] = math.inf
        got = run(dev, q, k, v, g, None, None)[3].double().cpu()
        assert bool((got[..., D - 2] == math.inf).all()), (sizes, D)
        rest = [c for c in range(D) if c != D - 2]
        check((got[..., rest],), (want[3][..., rest],), (bounds[3][..., rest],), f"{sizes} {D}")
