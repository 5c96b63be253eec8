"""packed_attention, forward and gradients, in calls of more than 2^22 scores whose sequences have more than 64 keys on the average: their bfloat16 kernels are others than those of
small calls (one term of the weights, tiles by 32-bit offsets).  Against the definition in float64, element by element (bounds: _packed.py): widths that fill their kernels and that
do not, keys in front of the queries, frames, shared heads whose rows do not divide a tile, walks that are shared, what is not to be read."""
import math

import pytest
import torch

from _packed import check, make, reference
from test_gpu_packed_attention import run

pytestmark = pytest.mark.gpu

SIZES = [
    # queries, keys (None: the same), query heads, key heads, causal, frame, tokens before, behind
    ([1900, 310, 0, 777], None, 2, 2, True, 1, 0, 0),
    ([1400, 130, 640], [2000, 990, 640], 3, 1, True, 1, 3, 70),
    ([1300, 700, 421], None, 5, 1, True, 54, 0, 0),
    ([2600], None, 1, 1, True, 1, 0, 0),                        # walks in pieces
    ([900, 350], [2100, 1650], 4, 2, True, 350, 129, 1),
    ([1500, 100], [2100, 60], 3, 3, False, 1, 0, 0),
    ([1700, 500], [900, 800], 6, 2, True, 1, 0, 5),             # rows without keys
    ([200] * 16, None, 8, 4, True, 1, 0, 0),
]


def few(lq, lk, hq):
    keys = sum(lk) // len(lk)
    return keys <= 64 or sum(lq) * hq <= (1 << 22) // keys


@pytest.mark.parametrize("D", [8, 24, 32, 40, 48, 56, 64, 72, 80, 88, 96, 104, 112, 120, 128])
@pytest.mark.parametrize("size", SIZES, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{c[2]}-{c[3]}-{c[4]}-{c[5]}")
def test_bfloat16(size, D, dev):
    lq, lk, hq, hkv, causal, frame, before, behind = size
    assert not few(lq, lk or lq, hq)
    print("packed_attention", size, D, flush=True)
    q, k, v, g, starts, key_starts = make(lq, lk or lq, hq, hkv, D, torch.bfloat16, sum(lq) + D, before, behind)
    want, bounds = reference(q, k, v, g, starts, key_starts, causal, frame)
    other = None if lk is None else key_starts
    got = run(dev, q, k, v, g, starts, other, causal, frame)
    check(got, want, bounds, f"{size} {D}")
    for a, b in zip(got, run(dev, q, k, v, g, starts, other, causal, frame)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D", [40, 64, 104, 128])
@pytest.mark.parametrize("garbage", [math.nan, math.inf, -math.inf, "lowest"])
def test_what_is_not_read_has_no_influence(garbage, D, dev):
    """Tokens at the beginning, in the middle and at the end of a sequence whose key, value, query and gradient of the output are no numbers: what does not read them, and what they do
    not read, as without them."""
    lq, lk, frame = [1500, 310], [1500, 900], 3
    assert not few(lq, lk, 4)
    q, k, v, g, starts, key_starts = make(lq, lk, 4, 2, D, torch.bfloat16, 9)
    want, bounds = reference(q, k, v, g, starts, key_starts, frame=frame)
    value = torch.finfo(torch.bfloat16).min if garbage == "lowest" else garbage
    for tokens in ([(0, 20), (1, 880)], [(0, 700), (1, 600)], [(0, 1480), (1, 895)]):      # sequence, token
        print("packed_attention", garbage, D, tokens, flush=True)
        fine = [torch.ones(t.shape[0], dtype=torch.bool) for t in (q, q, k, v)]
        dirty = [t.clone() for t in (q, k, v, g)]
        for s, token in tokens:
            row, key = int(starts[s]) + token - (lk[s] - lq[s]), int(key_starts[s]) + token
            dirty[0][row], dirty[1][key], dirty[2][key], dirty[3][row] = (value,) * 4
            first = token // frame * frame               # the first token that reads it
            for i in (0, 1):
                fine[i][int(starts[s]) + first - (lk[s] - lq[s]):int(starts[s + 1])] = False
            for i in (2, 3):
                fine[i][int(key_starts[s]):int(key_starts[s + 1])] = False
        check(run(dev, *dirty, starts, key_starts, frame=frame), want, bounds, f"{garbage} {tokens}", fine)
        # a gradient of the output alone, and a query alone: the keys' gradients behind what that token reads
        for which in (3, 0):
            dirty = [q, k, v, g]
            dirty[which] = dirty[which].clone()
            fine = [torch.ones(t.shape[0], dtype=torch.bool) for t in (q, q, k, v)]
            for s, token in tokens:
                row = int(starts[s]) + token - (lk[s] - lq[s])
                dirty[which][row] = value
                fine[1][row] = False
                if which == 0:
                    fine[0][row] = False
                for i in (2, 3):
                    fine[i][int(key_starts[s]):int(key_starts[s]) + token // frame * frame + frame] = False
            check(run(dev, *dirty, starts, key_starts, frame=frame), want, bounds, f"{which} {garbage} {tokens}", fine)


@pytest.mark.parametrize("D", [64, 128])
def test_infinities_that_are_read(D, dev):
    """An infinite value makes its channel infinite for those that read it, an infinite gradient of the output its channel of the values' gradient, and no other: where a token's tile
    has weights of one term, and of two."""
    for token in (3, 40, 700, 1490):
        q, k, v, g, starts, _ = make([1500, 90], [1500, 90], 4, 2, D, torch.bfloat16, 11)
        assert not few([1500, 90], [1500, 90], 4)
        v[token, 0, 5] = -math.inf
        want, bounds = reference(q, k, torch.where(v.isinf(), 0, v), g, starts, starts)
        out = run(dev, q, k, v, g, starts)[0].double().cpu()
        assert bool((out[token:1500, :2, 5] == -math.inf).all())
        free = torch.ones_like(out, dtype=torch.bool)
        free[token:1500, :2, 5] = False
        assert bool(((out - want[0]).abs() <= 1.05 * bounds[0] + 1e-30)[free].all())
        v[token, 0, 5], g[token, 1, 7] = 0.0, math.inf
        want, bounds = reference(q, k, v, torch.where(g.isinf(), 0, g), starts, starts)
        gv = run(dev, q, k, v, g, starts)[3].double().cpu()
        assert bool((gv[:token + 1, 0, 7] == math.inf).all())
        free = torch.ones_like(gv, dtype=torch.bool)
        free[:token + 1, 0, 7] = False
        assert bool(((gv - want[3]).abs() <= 1.05 * bounds[3] + 1e-30)[free].all())
