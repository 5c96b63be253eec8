"""Samples with one key that is to be read.  Its weight is 1, so gradients of queries and keys are 0 in exact arithmetic: exactly 0 in samples of up to 64 keys
(by their length), within the bounds of test_gpu_attention.py where a mask leaves one of more.  Where a number that they are made of is not finite, neither
are they 0: a weight of NaN (a score of NaN or +infinity), an infinite or undefined output, or such a gradient of it.  (A score of -infinity has no weight: a row
of no other is one without a key.)"""
import math

import pytest
import torch

from test_gpu_attention import check, make, reference, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Lk", [1, 50, 300])
@pytest.mark.parametrize("Lq", [1, 12, 70])
def test_undefined_numbers_leave_undefined_gradients(Lq, Lk, dtype, dev):
    """(in a row of the first sample; the second's are 0)"""
    lengths = torch.tensor([1, 1])
    for what, value in (("query", math.nan), ("query", math.inf), ("key", math.nan), ("value", math.nan), ("value", math.inf), ("grad", math.nan), ("grad", math.inf)):
        q, k, v, g = make(2, Lq, Lk, 4, 2, 40, dtype, 37)
        g[0, -1, 1, 3] = 2.0
        k[0, 0, 0, 3] = 1.5
        if what in ("query", "grad"):
            (q if what == "query" else g)[0, -1, 1, 3] = value
        else:
            (k if what == "key" else v)[0, 0, 0, 3] = value
        out, gq, gk, gv = run(dev, q, k, v, g, lengths, None)
        print(what, value, Lq, Lk, flush=True)
        rows = (slice(-1, None), slice(1, 2)) if what in ("query", "grad") else (slice(None), slice(0, 2))
        hit = gq[0][rows]
        if what == "query":
            assert bool(out[0][rows].isnan().all())
        assert bool(hit.isnan().all()), (what, value)
        clean = torch.ones_like(gq, dtype=torch.bool)
        clean[0][rows] = False
        assert not bool(gq[clean].any())
        assert bool(gk[0, 0, 0].isnan().all()), (what, value)
        assert not bool(gk[0, :, 1].any()) and not bool(gk[1].any()) and not bool(gk[0, 1:].any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("Lq", [1, 70, 2000])
def test_a_mask_that_leaves_one_key_of_many(Lq, dtype, dev):
    Lk = 300
    mask = torch.arange(Lk).expand(2, Lk) == torch.tensor([[200], [5]])
    q, k, v, g = make(2, Lq, Lk, 4, 2, 40, dtype, 41)
    want, bounds = reference(q, k, v, g, None, mask, 1.0 / math.sqrt(40))
    got = run(dev, q, k, v, g, None, mask)
    check(got, want, bounds, str(Lq))
    for n, key in enumerate((200, 5)):
        assert torch.equal(got[0][n].cpu(), v[n, key].repeat_interleave(2, 0).expand(Lq, 4, 40))


def test_a_long_sample_with_two_keys(dev):
    """bfloat16, two of 1000 keys that are to be read: weights of one term where the call is large, and of two where it is small; either within the bound"""
    for Lq in (70, 2500):
        q, k, v, g = make(2, Lq, 1000, 2, 1, 64, torch.bfloat16, 43)
        mask = torch.zeros(2, 1000, dtype=torch.bool)
        mask[0, 3], mask[0, 900], mask[1, 64], mask[1, 65] = True, True, True, True
        want, bounds = reference(q, k, v, g, None, mask, 1.0 / 8)
        check(run(dev, q, k, v, g, None, mask), want, bounds, str(Lq))
