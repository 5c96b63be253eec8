"""cross_attention with 2^26 rows and some: gradients of keys and values alone, whose delta is a launch of a wavefront to a row, are the sums of two halves'."""
import pytest
import torch

import d2conv3d_amd as d2c

pytestmark = pytest.mark.gpu


def test_gradients_of_keys_alone(dev):
    N, Lq, H, D, Lk = 2, (1 << 25) + 100, 1, 8, 5
    gen = torch.Generator(device=dev).manual_seed(3)
    q, g = (torch.randn(N, Lq, H, D, generator=gen, device=dev, dtype=torch.bfloat16) for _ in range(2))
    k, v = (torch.randn(N, Lk, H, D, generator=gen, device=dev, dtype=torch.bfloat16).requires_grad_() for _ in range(2))
    print("cross_attention", q.shape, flush=True)
    got = torch.autograd.grad(d2c.cross_attention(q, k, v), (k, v), g)
    half = Lq // 2
    parts = [torch.autograd.grad(d2c.cross_attention(q[:, s], k, v), (k, v), g[:, s]) for s in (slice(0, half), slice(half, Lq))]
    for a, b, c in zip(got, *parts):
        want = b.double() + c.double()
        # (each of the three is rounded to bfloat16, and a sum of 2^25 terms of either sign has errors of its own: 2^-24 of it to a tile of 64 rows at most)
        bound = 2.0 ** -8 * (a.double().abs() + b.double().abs() + c.double().abs()) + 2.0 ** -24 * Lq / 64 * 8
        assert bool(((a.double() - want).abs() <= bound).all()), ((a.double() - want).abs() / bound).max()
