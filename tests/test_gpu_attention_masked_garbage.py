"""What keys and values hold that are not to be read has no influence, for every width and both lines of the backward pass: infinities of both signs, NaN and
the type's lowest value planted among those that are read, outputs and gradients to the bit."""
import math

import pytest
import torch

from test_gpu_attention import make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [8, 24, 33, 40, 56, 72, 80, 96, 104, 112, 120, 127, 128])
def test_garbage(D, dtype, dev):
    print("cross_attention, garbage in masked keys", D, dtype, flush=True)
    for N, Lq, Lk, Hq, Hkv in ((2, 1, 300, 4, 2), (2, 9, 700, 2, 1), (2, 70, 333, 2, 1), (2, 40, 60, 2, 2), (2, 600, 1000, 4, 2)):
        q, k, v, g = make(N, Lq, Lk, Hq, Hkv, D, dtype, D + Lk)
        gen = torch.Generator().manual_seed(D)
        mask = torch.rand(N, Lk, generator=gen) < 0.6
        lengths = torch.tensor([Lk, Lk - 20])
        hidden = ~(mask & (torch.arange(Lk) < lengths[:, None]))
        want = run(dev, q, k, v, g, lengths, mask)
        garbage = torch.tensor([math.inf, -math.inf, math.nan, torch.finfo(dtype).min])
        for t in (k, v):
            what = garbage[torch.randint(0, 4, t.shape, generator=gen)].to(dtype)
            t[hidden] = what[hidden]
        for a, b in zip(run(dev, q, k, v, g, lengths, mask), want):
            assert torch.equal(a, b) and not bool(a.isnan().any()), (N, Lq, Lk, D)
