"""packed_attention, bfloat16: sums of 64 terms or fewer have weights of two terms whatever they are packed with, so that rows that read few keys, the gradients of
keys that few rows read, and whole short sequences are off by float32 arithmetic and the rounding of the result alone.

Bounds: the first term is cut off, not rounded (what is left is below 2^-7 of the weight), the second a bfloat16 of that, off by 2^-8 of it: 2^-15 of a weight.  ds, whose first
term is rounded (2^-8): 2^-16.  delta: the output before it is rounded (2^-15 A and float32 arithmetic) but for the rounding of what rounding takes from it, 2^-16 of it.  Each result is
rounded once, u = 2^-8.  float32: E as in _packed.py."""
import math

import pytest
import torch

from _packed import U16, U32, allowed, make
from test_gpu_packed_attention import run

CASES = [
    # queries, keys (None: the same), query heads, key heads, causal, frame
    ([2950, 2, 3, 1, 40, 64, 17, 4], None, 4, 2, True, 1),
    ([2, 5, 1, 2, 3200, 3, 2], None, 3, 1, True, 1),
    ([1200, 3, 12, 2], [3500, 3, 20, 300], 4, 4, True, 1),
    ([1500, 24, 6, 1100], None, 6, 2, True, 6),
    ([2700, 2, 2, 60, 1], [2700, 2, 4, 64, 2], 3, 3, False, 1),
    ([2600, 30, 3], [1700, 10, 2], 4, 2, True, 1),             # queries in front of their keys
]


def definition(q, k, v, g, starts, key_starts, causal, frame, one_term=False):
    """Per result (out and the gradients): its value, the bound of what has two terms, which elements that is, and, `one_term`, what weights of one term would make of it."""
    T, hq, D = q.shape
    rep, scale = hq // k.shape[1], 1.0 / math.sqrt(D)
    likes = (q, q, k, v)
    value, bound, other = ([torch.zeros(t.shape, dtype=torch.float64) for t in likes] for _ in range(3))
    which = [torch.zeros(t.shape[:2], dtype=torch.bool) for t in likes]

    def rounded(t):
        return t.float().bfloat16().double()
    for s in range(len(starts) - 1):
        rows, keys = slice(int(starts[s]), int(starts[s + 1])), slice(int(key_starts[s]), int(key_starts[s + 1]))
        lq, lk = rows.stop - rows.start, keys.stop - keys.start
        if lq == 0 or lk == 0:
            continue
        ok = allowed(lq, lk, causal, frame)
        few_keys, few_rows = ok.sum(1) <= 64, ok.sum(0) * rep <= 64
        for h in range(hq):
            Q, G, K, V = q[rows, h].double(), g[rows, h].double(), k[keys, h // rep].double(), v[keys, h // rep].double()
            sabs = (Q.abs() @ K.abs().t()) * scale
            score = ((Q @ K.t()) * scale).masked_fill(~ok, -math.inf)
            top = score.amax(-1, keepdim=True)
            w = torch.exp(score - torch.where(top.isinf(), 0.0, top))
            total = w.sum(-1, keepdim=True).clamp_min(1e-300)
            p = w / total
            out, A = p @ V, p @ V.abs()
            one = ok.sum(-1, keepdim=True) == 1
            dp, delta = G @ V.t(), (G * out).sum(-1, keepdim=True)
            ds = torch.where(one, 0.0, p * (dp - delta))
            E = U32 * (D + 64 + max(lq * rep, lk) / 8 + 4 * sabs.max().item())
            pabs = torch.where(one, 0.0, p * (G.abs() @ V.abs().t() + (G.abs() * A).sum(-1, keepdim=True)))
            eds = torch.where(one, 0.0, 2.0 ** -16 * ds.abs() + p * (G.abs() * ((2.0 ** -15 + 2 * E) * A + 2.0 ** -16 * out.abs())).sum(-1, keepdim=True) + 4 * E * pabs)
            parts = ((rows, h, out, (2.0 ** -15 + 2 * E) * A, few_keys),
                     (rows, h, ds @ K * scale, (eds @ K.abs() + 2 * E * (pabs @ K.abs())) * scale, few_keys),
                     # (delta of its rows is that of two terms, too)
                     (keys, h // rep, ds.t() @ Q * scale, (eds.t() @ Q.abs() + 2 * E * (pabs.t() @ Q.abs())) * scale, few_rows & few_keys.all()),
                     (keys, h // rep, p.t() @ G, (2.0 ** -15 + 2 * E) * (p.t() @ G.abs()), few_rows))
            for i, (at, head, x, b, some) in enumerate(parts):
                value[i][at, head] += x
                bound[i][at, head] += b
                which[i][at, head] = some
            if one_term:
                ds1 = rounded(ds)
                for i, (at, head, x) in enumerate(((rows, h, rounded(w) @ V / total), (rows, h, ds1 @ K * scale), (keys, h // rep, ds1.t() @ Q * scale), (keys, h // rep, rounded(p).t() @ G))):
                    other[i][at, head] += x
    for i in range(4):
        bound[i] += U16 * value[i].abs()
    return value, bound, which, [rounded(t) for t in other]


def inputs(case, D):
    lq, lk, hq, hkv, causal, frame = case
    assert sum(lq) * hq * (sum(lk or lq) // len(lq)) > 1 << 22 and sum(lk or lq) // len(lq) > 64      # (on the kernels of one term)
    return make(lq, lk or lq, hq, hkv, D, torch.bfloat16, sum(lq) + D), causal, frame


NAMES = ("out", "grad_query", "grad_key", "grad_value")


@pytest.mark.gpu
@pytest.mark.parametrize("D", [24, 40, 64, 80, 104, 128])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{c[2]}-{c[3]}-{c[4]}-{c[5]}")
def test_two_terms(case, D, dev):
    print("packed_attention", case, D, flush=True)
    (q, k, v, g, starts, key_starts), causal, frame = inputs(case, D)
    value, bound, which, _ = definition(q, k, v, g, starts, key_starts, causal, frame)
    got = run(dev, q, k, v, g, starts, None if case[1] is None else key_starts, causal, frame)
    for name, a, e, b, some in zip(NAMES, got, value, bound, which):
        assert bool(some.any()), name
        over = ((a.detach().double().cpu() - e).abs() / (1.05 * b + 1e-30))[some]
        bad = ~(over <= 1.0)
        assert not bool(bad.any()), f"{name}: {int(bad.sum())} of {over.numel()} beyond the bound, worst {over.max().item():.2f} of it"


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{c[2]}-{c[3]}-{c[4]}-{c[5]}")
def test_the_bounds_tell_one_term(case):
    """(the definition alone, on the CPU)"""
    (q, k, v, g, starts, key_starts), causal, frame = inputs(case, 64)
    value, bound, which, other = definition(q, k, v, g, starts, key_starts, causal, frame, True)
    for name, e, b, some, x in zip(NAMES, value, bound, which, other):
        over = ((x - e).abs() / (1.05 * b + 1e-30))[some]
        assert bool((over > 1.0).any()), (name, over.max().item())
        print(name, int((over > 1.0).sum()), "of", over.numel(), "beyond the bound, worst", round(over.max().item(), 2))
