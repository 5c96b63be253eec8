"""Room for partial sums of cross_attention: how much a call asks for at most, and calls that run without where the GPU's memory does not have it."""
import contextlib
import ctypes
import math

import pytest
import torch

import d2conv3d_amd as d2c
from d2conv3d_amd import _lib, attention
from test_gpu_attention import check, make, reference

pytestmark = pytest.mark.gpu

PART_BYTES = 256 << 20


def desc(N, Lq, Lk, Hq, Hkv, D, dtype, part_limit=0):
    l3 = ctypes.c_int64 * 3
    q, k = (l3(n * h * D, h * D, D) for n, h in ((Lq, Hq), (Lk, Hkv)))
    return _lib.AttentionDesc(N=N, Lq=Lq, Lk=Lk, Hq=Hq, Hkv=Hkv, D=D, dtype=dtype, scale=0.1, q_stride=q, k_stride=k, v_stride=k,
                              part_limit=part_limit)


@pytest.mark.parametrize("dtype", [0, 2])
def test_what_a_call_asks_for_at_most(dtype, dev):
    lib = _lib.load()
    fwd, bwd = lib.d2c_attention_forward_workspace_bytes, lib.d2c_attention_backward_workspace_bytes
    shared = 0
    for heads in (1, 3, 8, 40):
        for Lq in (1, 20, 777, 9000, 40000):
            for Lk in (100, 5000, 1 << 20, 1 << 24):
                for D in (33, 64, 128):
                    size = heads, Lq, Lk, heads, heads, D, dtype
                    delta = (heads * heads * Lq * 4 + 255) // 256 * 256
                    for limit, most in ((0, PART_BYTES), (1 << 20, 1 << 20), (-1, 0)):
                        q = desc(*size, part_limit=limit)
                        room = 512 if most else 0                   # (rounded up)
                        assert fwd(ctypes.byref(q)) <= most + room, (size, limit)
                        assert bwd(ctypes.byref(q)) <= delta + most + room, (size, limit)
                        shared = max(shared, fwd(ctypes.byref(q)))
    assert shared > 1 << 20


@contextlib.contextmanager
def no_room_beyond(room, dev):
    """The allocator gets `room` more bytes than it has reserved; nothing freed is kept."""
    torch.cuda.synchronize(dev)
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(dev).total_memory
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved(dev) + room) / total, dev)
    try:
        yield
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0, dev)
        torch.cuda.synchronize(dev)
        torch.cuda.empty_cache()


@pytest.mark.parametrize("route", ["native", "python"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_room_for_them(dtype, route, dev, monkeypatch):
    if route == "python":
        monkeypatch.setattr(attention, "_try_native", lambda *a: None)
        monkeypatch.setattr("d2conv3d_amd._ops._WS_CACHE_ON", [False])
    N, Lq, Lk, H, D = 1, 260, 20000, 4, 128
    lib = _lib.load()
    code = 2 if dtype == torch.bfloat16 else 0
    room = 6 << 20
    q = desc(N, Lq, Lk, H, H, D, code)
    assert lib.d2c_attention_forward_workspace_bytes(ctypes.byref(q)) > room
    q, k, v, g = make(N, Lq, Lk, H, H, D, dtype, 5)
    want, bounds = reference(q, k, v, g, None, None, 1.0 / math.sqrt(D))
    args = [t.to(dev).requires_grad_() for t in (q, k, v)]
    g = g.to(dev)
    with no_room_beyond(room, dev):                    # (output, low and sums of the rows: 1 MB, in pools of 2 MB)
        out = d2c.cross_attention(*args)
    check((out, *torch.autograd.grad(out, args, g)), want, bounds, f"{dtype} {route}")
    k, v = (t.detach() for t in args[1:])              # (their gradients are 20 to 40 MB each)
    out = d2c.cross_attention(args[0], k, v)
    with no_room_beyond(room, dev):
        (alone,) = torch.autograd.grad(out, args[:1], g)
    check((out, alone), want[:2], bounds[:2], f"{dtype} {route}")
