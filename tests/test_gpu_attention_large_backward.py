"""Gradients of cross_attention in calls of more than 2^22 scores, whose bfloat16 kernels are others than those of small calls (one term of the weights, tiles
by 32-bit offsets), against the definition in float64, element by element: widths that fill their kernels and that do not, frames that are not to be read,
lengths, shared heads, tiles that end inside.  Bounds: test_gpu_attention.py."""
import math

import pytest
import torch

from test_gpu_attention import check, make, make_masks, reference, run

pytestmark = pytest.mark.gpu

SIZES = [
    # N, Lq, Lk, Hq, Hkv, mask
    (1, 1100, 2000, 2, 2, "none"),
    (2, 530, 1030, 4, 2, "frames"),
    (3, 333, 2150, 2, 1, "lengths"),
    (2, 150, 3600, 4, 4, "both"),
    (1, 9000, 520, 1, 1, "frames"),
]


def masks(kind, N, Lk):
    if kind != "frames":
        return make_masks(kind, N, Lk, 7)
    keep = torch.rand(N, 16, generator=torch.Generator().manual_seed(7)) < 0.7
    keep[:, 3] = False                           # (whole tiles without a key)
    return None, keep[:, torch.arange(Lk) * 16 // Lk].contiguous()


@pytest.mark.parametrize("D", [24, 32, 40, 56, 64, 72, 80, 96, 104, 120, 128])
@pytest.mark.parametrize("size", SIZES)
def test_bfloat16(size, D, dev):
    *sizes, kind = size
    N, Lq, Lk, Hq, _ = sizes
    assert N * Lq * Lk * Hq > 1 << 22 and Lk > 64
    print("cross_attention", size, D, flush=True)
    q, k, v, g = make(*sizes, D, torch.bfloat16, seed=sum(sizes) + D)
    lengths, mask = masks(kind, N, Lk)
    want, bounds = reference(q, k, v, g, lengths, mask, 1.0 / math.sqrt(D))
    got = run(dev, q, k, v, g, lengths, mask)
    check(got, want, bounds, f"{size} {D}")
    for a, b in zip(got, run(dev, q, k, v, g, lengths, mask)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D", [40, 64, 128])
def test_float32(D, dev):
    for size in SIZES[:3]:
        *sizes, kind = size
        q, k, v, g = make(*sizes, D, torch.float32, seed=sum(sizes) + D)
        lengths, mask = masks(kind, sizes[0], sizes[2])
        want, bounds = reference(q, k, v, g, lengths, mask, 1.0 / math.sqrt(D))
        check(run(dev, q, k, v, g, lengths, mask), want, bounds, f"{size} {D}")
