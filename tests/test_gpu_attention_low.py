"""What rounding takes from bfloat16 outputs of cross_attention and is kept for the gradients: it is there on every route of the forward pass, and
delta = sum_d do o is that of the output before it was rounded.

Queries of 0 give every key that is there the weight 1 / keys, a sum of which is exact in float32 before it is divided; so the output before it is rounded
is off by float32 arithmetic alone, E = u32 (D + 64 + keys / 8) mean |v|, and output + low by 2^-16 |o| more (low is a bfloat16 of at most 2^-8 |o|, off by
2^-8 of itself).

Gradients of the queries: gq = scale sum_j ds_j k_j, ds_j = (do (v_j - o)) / keys, rounded to bfloat16 (2^-8 |ds_j| each at most), with delta off by
sum |do| (2^-16 |o| + 2 E), then rounded (2^-8 |gq|).  Values far from 0 (mean 64.2, between two bfloat16 numbers 0.5 apart) beside keys far from 0 (mean 4) make an error of delta, which is the
same for all keys, many times what the other roundings add up to: delta made of the rounded output would be off by up to 2^-8 |o| |do| a channel."""
import contextlib
import math

import pytest
import torch

import d2conv3d_amd as d2c
from d2conv3d_amd import attention

pytestmark = pytest.mark.gpu

U32, U16 = 2.0 ** -24, 2.0 ** -8


def case(N, Lq, Lk, Hq, Hkv, D, seed):
    gen = torch.Generator().manual_seed(seed)

    def rn(*s):
        return torch.randn(*s, generator=gen)
    return (torch.zeros(N, Lq, Hq, D).bfloat16(), (rn(N, Lk, Hkv, D) + 4).bfloat16(), (rn(N, Lk, Hkv, D) + 64.2).bfloat16(),
            rn(N, Lq, Hq, D).bfloat16())


def definition(k, v, g, ok, Hq, scale, ds_u):
    """(out, its float32 error, gq, its bound) in float64; ok [N, Lk]"""
    N, Lk, Hkv, D = k.shape
    rep = Hq // Hkv
    K, V = (t.double().repeat_interleave(rep, 2).permute(0, 2, 1, 3) for t in (k, v))      # [N, Hq, Lk, D]
    G = g.double().permute(0, 2, 1, 3)
    w = (ok.double() / ok.sum(1, keepdim=True).clamp_min(1))[:, None, :, None]
    o = (w * V).sum(2, keepdim=True).expand(-1, -1, G.size(2), -1)
    E = U32 * (D + 64 + Lk / 8) * (w * V.abs()).sum(2, keepdim=True)
    dp = G @ V.transpose(-1, -2).contiguous()
    delta = (G * o).sum(-1, keepdim=True)
    p = w.transpose(-1, -2)
    ds = p * (dp - delta)
    off = (G.abs() * (2.0 ** -16 * o.abs() + 2 * E)).sum(-1, keepdim=True)                  # of delta
    e32 = 2 * U32 * (D + 64 + Lk / 8) * (G.abs() @ V.abs().transpose(-1, -2).contiguous())        # of dp
    eds = ds_u * ds.abs() + p * (off + e32)
    gq = ds @ K * scale
    bound = eds @ K.abs() * scale + U16 * gq.abs()
    return [t.permute(0, 2, 1, 3) for t in (o, E.expand_as(o), gq, bound)]


CASES = [
    # N, Lq, Lk, Hq, Hkv, D, masked
    (1, 1, 3000, 4, 1, 64, False),       # up to 8 rows of a key head; keys shared by workgroups
    (2, 2, 200, 2, 1, 40, True),
    (1, 20, 3000, 1, 1, 64, False),      # up to 32
    (2, 11, 300, 4, 2, 104, True),
    (1, 200, 300, 2, 2, 64, True),       # more
    (1, 300, 9000, 2, 1, 64, False),     # ... more than 2^22 scores, walks shared
    (1, 300, 9000, 2, 1, 128, True),
    (2, 3000, 400, 2, 2, 40, True),
    (1, 50, 300, 2, 1, 33, False),       # heads of an odd size
    (2, 50, 60, 2, 1, 64, True),         # few keys
    (1, 3, 30, 2, 2, 64, False),
]


@contextlib.contextmanager
def python_route():
    with pytest.MonkeyPatch.context() as mp:
        mp.setattr(attention, "_try_native", lambda *a: None)
        yield


def inputs(args, dev):
    N, Lq, Lk, Hq, Hkv, D, masked = args
    q, k, v, g = case(N, Lq, Lk, Hq, Hkv, D, Lq + Lk + D)
    mask = torch.rand(N, Lk, generator=torch.Generator().manual_seed(3)) < 0.6 if masked else None
    ok = torch.ones(N, Lk, dtype=torch.bool) if mask is None else mask
    return [t.to(dev) for t in (q, k, v, g)], None if mask is None else mask.to(dev), (k, v, g, ok, Hq, 1.0 / math.sqrt(D))


@pytest.mark.parametrize("args", CASES)
def test_output_and_low_are_the_output_before_it_is_rounded(args, dev):
    print("cross_attention, out_low", args, flush=True)
    (q, k, v, g), mask, plain = inputs(args, dev)
    o, E, _, _ = definition(*plain, 0.0)
    with python_route():
        out = d2c.cross_attention(q.requires_grad_(), k, v, key_mask=mask)
        low = out.grad_fn.saved_tensors[6]
    assert low.shape == out.shape and low.dtype == torch.bfloat16
    whole = (out.detach().double() + low.double()).cpu()
    over = (whole - o).abs() / (1.05 * (E + 2.0 ** -16 * o.abs()))
    assert not bool((~(over <= 1.0)).any()), f"worst {over.max().item():.2f} of the bound"


@pytest.mark.parametrize("route", ["native", "python"])
@pytest.mark.parametrize("args", CASES)
def test_delta_is_that_of_the_output_before_it_is_rounded(args, route, dev):
    (q, k, v, g), mask, plain = inputs(args, dev)
    _, _, want, bound = definition(*plain, U16)
    with python_route() if route == "python" else contextlib.nullcontext():
        q.requires_grad_()
        (gq,) = torch.autograd.grad(d2c.cross_attention(q, k, v, key_mask=mask), q, g)
    over = (gq.double().cpu() - want).abs() / (1.05 * bound + 1e-30)
    assert not bool((~(over <= 1.0)).any()), f"worst {over.max().item():.2f} of the bound, {int((~(over <= 1.0)).sum())} of {over.numel()}"


def test_the_bound_tells_a_delta_of_the_rounded_output():
    """(the definition alone, on the CPU)"""
    for args in CASES:
        _, _, plain = inputs(args, "cpu")
        o, _, want, bound = definition(*plain, U16)
        k, v, g, ok, Hq, scale = plain
        K, V = (t.double().repeat_interleave(Hq // k.size(2), 2).permute(0, 2, 1, 3) for t in (k, v))
        G, O = g.double().permute(0, 2, 1, 3), o.permute(0, 2, 1, 3).bfloat16().double()
        p = (ok.double() / ok.sum(1, keepdim=True))[:, None, None, :]
        ds = p * (G @ V.transpose(-1, -2).contiguous() - (G * O).sum(-1, keepdim=True))
        off = (ds @ K * scale).permute(0, 2, 1, 3)
        assert float(((off - want).abs() / bound).max()) > 2.0, args
