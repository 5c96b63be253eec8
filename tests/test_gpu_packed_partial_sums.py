"""Room for partial sums of packed_attention: how much a call asks for at most, and calls that run without where the GPU's memory does not have it."""
import ctypes

import pytest
import torch

import d2conv3d_amd as d2c
from _packed import check, make, reference
from d2conv3d_amd import _lib, attention
from test_gpu_attention_partial_sums import PART_BYTES, no_room_beyond

pytestmark = pytest.mark.gpu


def desc(sequences, queries, keys, Hq, Hkv, D, dtype, causal=1, part_limit=0):
    l2 = ctypes.c_int64 * 2
    q, k = (l2(h * D, D) for h in (Hq, Hkv))
    return _lib.PackedAttentionDesc(sequences, Hq, Hkv, D, dtype, causal, 1, 0.1, queries, keys, q, k, k, part_limit)


@pytest.mark.parametrize("dtype", [0, 2])
def test_what_a_call_asks_for_at_most(dtype, dev):
    lib = _lib.load()
    fwd, bwd = lib.d2c_packed_attention_forward_workspace_bytes, lib.d2c_packed_attention_backward_workspace_bytes
    shared = [0, 0]
    for sequences in (1, 3, 200):
        for heads in (1, 8, 40):
            for queries, keys in ((1, 1 << 24), (300, 5000), (40000, 40000), (40000, 1 << 20), (1 << 20, 1 << 20), (1 << 22, 100)):
                for D in (33, 64, 128):
                    size = sequences, queries, keys, heads, heads, D, dtype
                    delta = queries * heads * 4
                    for limit, most in ((0, PART_BYTES), (1 << 20, 1 << 20), (-1, 0)):
                        q = desc(*size, part_limit=limit)
                        asked = fwd(ctypes.byref(q)), bwd(ctypes.byref(q)) - delta
                        assert asked[0] <= most + 512 and 0 <= asked[1] <= most + 512, (size, limit, asked)      # (rounded up)
                        shared = [max(x) for x in zip(shared, asked)]
    assert min(shared) > 1 << 20


@pytest.mark.parametrize("route", ["native", "python"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lq,lk,causal", [([260], [20000], True), ([20000], [200], False)])
def test_no_room_for_them(lq, lk, causal, dtype, route, dev, monkeypatch):
    if route == "python":
        monkeypatch.setattr(attention, "_try_native", lambda *a: None)
        monkeypatch.setattr("d2conv3d_amd._ops._WS_CACHE_ON", [False])
    H, D, room = 4, 128, 6 << 20
    q, k, v, g, starts, key_starts = make(lq, lk, H, H, D, dtype, 5)
    asked = [size(ctypes.byref(desc(1, lq[0], lk[0], H, H, D, 2 if dtype == torch.bfloat16 else 0, int(causal))))
             for size in (_lib.load().d2c_packed_attention_forward_workspace_bytes, _lib.load().d2c_packed_attention_backward_workspace_bytes)]
    want, bounds = reference(q, k, v, g, starts, key_starts, causal)
    args = [t.to(dev).requires_grad_() for t in (q, k, v)]
    g, starts, key_starts = (t.to(dev) for t in (g, starts, key_starts))
    few_rows = lq[0] < lk[0]      # (what is as long as 20000 tokens has no room either)
    assert asked[0 if few_rows else 1] > room
    if few_rows:
        with no_room_beyond(room, dev):
            out = d2c.packed_attention(*args, starts, key_starts, causal)
        check((out, *torch.autograd.grad(out, args, g)), want, bounds, f"{dtype} {route}")
    else:
        args[0], args[2] = args[0].detach(), args[2].detach()
        out = d2c.packed_attention(*args, starts, key_starts, causal)
        with no_room_beyond(room, dev):
            (alone,) = torch.autograd.grad(out, args[1:2], g)
        check((out,), want[:1], bounds[:1], f"{dtype} {route}")
        check((alone,), want[2:3], bounds[2:3], f"{dtype} {route}")
