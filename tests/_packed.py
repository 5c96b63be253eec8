"""Attention inside packed sequences in float64, sequence by sequence, with the bounds of the types' errors.

u = the unit roundoff, 2^-8 for bfloat16; A = sum_j p_j |v_j| and its like for the gradients.  bfloat16 rounds the weights p (and ds) to the
matrix instruction's operands and the result once, u each, so an output is off by 2 u A; float32 arithmetic adds E = u32 (D + 64 + L / 8 + 4 max_s) A,
L the length of the sum: products and sums over D channels and L positions, and an exponential whose argument of size max_s is rounded."""
import math

import torch

U32, U16 = 2.0 ** -24, 2.0 ** -8


def make(lq, lk, hq, hkv, D, dtype, seed, before=0, behind=0):
    """(q, k, v, grad_out, starts, key_starts), `before` and `behind`: tokens of no sequence"""
    gen = torch.Generator().manual_seed(seed)
    T, Tk = (before + sum(x) + behind for x in (lq, lk))

    def rn(*shape):
        return torch.randn(*shape, generator=gen).to(dtype)
    starts, key_starts = (torch.tensor([before] + x).cumsum(0).int() for x in (lq, lk))
    return rn(T, hq, D), rn(Tk, hkv, D), rn(Tk, hkv, D), rn(T, hq, D), starts, key_starts


def allowed(lq, lk, causal, frame):
    if not causal:
        return torch.ones(lq, lk, dtype=torch.bool)
    token = torch.arange(lq) + lk - lq
    return torch.div(torch.arange(lk), frame, rounding_mode="floor")[None] <= torch.div(token, frame, rounding_mode="floor")[:, None]


def reference(q, k, v, g, starts, key_starts, causal=True, frame=1, scale=None):
    """((out, gq, gk, gv), their bounds)"""
    u = U16 if q.dtype == torch.bfloat16 else 0.0
    T, hq, D = q.shape
    rep = hq // k.shape[1]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    results = [torch.zeros(t.shape, dtype=torch.float64) for t in (q, q, k, v)]
    bounds = [torch.zeros(t.shape, dtype=torch.float64) for t in (q, q, k, v)]
    for s in range(len(starts) - 1):
        rows, keys = slice(int(starts[s]), int(starts[s + 1])), slice(int(key_starts[s]), int(key_starts[s + 1]))
        lq, lk = rows.stop - rows.start, keys.stop - keys.start
        if lq == 0 or lk == 0:
            continue
        ok = allowed(lq, lk, causal, frame)
        for h in range(hq):
            Q, G, K, V = q[rows, h].double(), g[rows, h].double(), k[keys, h // rep].double(), v[keys, h // rep].double()
            sabs = (Q.abs() @ K.abs().t()) * scale
            score = ((Q @ K.t()) * scale).masked_fill(~ok, -math.inf)
            top = score.amax(-1, keepdim=True)
            e = torch.exp(score - torch.where(top.isinf(), 0.0, top))
            p = e / e.sum(-1, keepdim=True).clamp_min(1e-300)
            out = p @ V
            delta = (G * out).sum(-1, keepdim=True)
            one = ok.sum(-1, keepdim=True) == 1      # (exact zeros)
            ds = torch.where(one, 0.0, p * (G @ V.t() - delta))
            e32 = U32 * (D + 64 + max(lq * rep, lk) / 8 + 4 * sabs.max().item())
            A = p @ V.abs()
            b_out = 2 * (u + e32) * A
            pabs = p * (G.abs() @ V.abs().t() + (G.abs() * A).sum(-1, keepdim=True))
            # (what rounding takes off the output is kept for delta)
            eds = torch.where(one, 0.0, u * ds.abs() + p * (G.abs() * (u + 2 * e32) * A).sum(-1, keepdim=True) + 4 * e32 * pabs)
            pabs = torch.where(one, 0.0, pabs)
            for i, (at, x, b) in enumerate(((slice(None), out, b_out), (slice(None), ds @ K * scale, (eds @ K.abs() + 2 * e32 * (pabs @ K.abs())) * scale),
                                            (None, ds.t() @ Q * scale, (eds.t() @ Q.abs() + 2 * e32 * (pabs.t() @ Q.abs())) * scale),
                                            (None, p.t() @ G, (u + 2 * e32) * (p.t() @ G.abs())))):
                where = (rows, h) if at is not None else (keys, h // rep)
                results[i][where] += x
                bounds[i][where] += b
    for i in (1, 2, 3):
        bounds[i] += u * results[i].abs()
    return results, bounds


def check(got, want, bounds, what="", where=(None,) * 4):
    for name, a, e, b, at in zip(("out", "grad_query", "grad_key", "grad_value"), got, want, bounds, where):
        a = a.detach().double().cpu()
        assert a.shape == e.shape, (what, name, a.shape, e.shape)
        over = (a - e).abs() / (1.05 * b + 1e-30)
        if at is not None:
            over = over[at]
        bad = ~(over <= 1.0)
        assert not bool(bad.any()), f"{what} {name}: {int(bad.sum())} of {over.numel()} beyond the bound, worst {over.max().item():.2f} of it, NaN {int(over.isnan().sum())}"
