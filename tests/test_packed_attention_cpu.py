"""What packed_attention refuses, and what it asks for, without a GPU."""
import ctypes
import math

import pytest
import torch

import d2conv3d_amd as d2c
from d2conv3d_amd import _lib


def desc(**kw):
    base = dict(sequences=2, Hq=4, Hkv=2, D=64, dtype=0, causal=1, frame=1, scale=0.125, queries=100, keys=100)
    base.update(kw)
    strides = [(ctypes.c_int64 * 2)(base["Hq"] * base["D"], base["D"])] + [(ctypes.c_int64 * 2)(base["Hkv"] * base["D"], base["D"])] * 2
    return _lib.PackedAttentionDesc(*base.values(), *strides)


@pytest.mark.parametrize("change,message", [
    (dict(dtype=1), "float32 or bfloat16"), (dict(sequences=-1), "negative"), (dict(queries=-1), "negative"), (dict(keys=-1), "negative"), (dict(Hq=0), "positive"),
    (dict(Hkv=0), "positive"), (dict(D=0), "positive"), (dict(Hq=3), "multiple"), (dict(D=136), "128"), (dict(frame=0), "frame"), (dict(frame=-4), "frame"),
    (dict(frame=(1 << 30) + 1), "frame"), (dict(scale=0.0), "scale"), (dict(scale=math.inf), "scale"), (dict(scale=math.nan), "scale"),
    (dict(queries=1 << 30), "too many"), (dict(queries=1 << 29), "too many"), (dict(keys=1 << 30), "too many"), (dict(sequences=1 << 20), "too many"), (dict(Hq=1 << 20, Hkv=1 << 20), "too many")])
def test_descriptions_that_are_refused(change, message):
    lib = _lib.load()
    q = desc(**change)
    assert lib.d2c_packed_attention_forward(ctypes.byref(q), *(None,) * 9, 0, None) != 0 and message in _lib.last_error()
    assert lib.d2c_packed_attention_backward(ctypes.byref(q), *(None,) * 13, 0, None) != 0 and message in _lib.last_error()
    assert lib.d2c_packed_attention_forward_workspace_bytes(ctypes.byref(q)) == 0 and lib.d2c_packed_attention_backward_workspace_bytes(ctypes.byref(q)) == 0


def test_calls_that_are_refused():
    lib = _lib.load()
    some = ctypes.c_void_p(4096)
    assert lib.d2c_packed_attention_forward(ctypes.byref(desc()), *(None,) * 9, 0, None) != 0 and "null" in _lib.last_error()
    assert lib.d2c_packed_attention_backward(ctypes.byref(desc()), *(None,) * 13, 0, None) != 0 and "null" in _lib.last_error()
    nb = lib.d2c_packed_attention_backward_workspace_bytes(ctypes.byref(desc()))
    assert nb >= 100 * 4 * 4
    for ws, have in ((None, 0), (ctypes.c_void_p(1 << 20), nb - 1), (ctypes.c_void_p((1 << 20) + 16), nb)):
        assert lib.d2c_packed_attention_backward(ctypes.byref(desc()), *(some,) * 12, ws, have, None) != 0 and "workspace" in _lib.last_error()
    q = desc(queries=0, keys=0)
    assert lib.d2c_packed_attention_forward(ctypes.byref(q), *(None,) * 9, 0, None) == 0 and lib.d2c_packed_attention_backward(ctypes.byref(q), *(None,) * 13, 0, None) == 0


class OnTheGpu(torch.Tensor):
    """A CPU tensor that says it is on the GPU: what the argument checks look at, with no memory touched."""
    is_cuda = True


def gpu(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnTheGpu)


STARTS = torch.tensor([0, 4, 6]).as_subclass(OnTheGpu)


@pytest.mark.parametrize("args,kw,message", [
    ((gpu(6, 2, 16, 1), gpu(6, 1, 16), gpu(6, 1, 16), STARTS), {}, "dimensions"),
    ((gpu(6, 2, 16), gpu(6, 1, 16), gpu(6, 2, 16), STARTS), {}, "differ in shape"),
    ((gpu(6, 2, 16), gpu(6, 1, 8), gpu(6, 1, 8), STARTS), {}, "does not fit"),
    ((gpu(6, 3, 16), gpu(6, 2, 16), gpu(6, 2, 16), STARTS), {}, "multiple"),
    ((gpu(6, 2, 130), gpu(6, 1, 130), gpu(6, 1, 130), STARTS), {}, "128 channels"),
    ((gpu(6, 2, 16), gpu(6, 1, 16).double(), gpu(6, 1, 16), STARTS), {}, "one dtype"),
    ((gpu(6, 2, 16), gpu(7, 1, 16), gpu(7, 1, 16), STARTS), {}, "as many keys"),
    ((gpu(6, 2, 16), gpu(6, 1, 16), gpu(6, 1, 16), gpu(3)), {}, "whole numbers"),
    ((gpu(6, 2, 16), gpu(6, 1, 16), gpu(6, 1, 16), gpu(0, dtype=torch.int32)), {}, "whole numbers"),
    ((gpu(6, 2, 16), gpu(6, 1, 16), gpu(6, 1, 16), STARTS, STARTS[:2]), {}, "key_starts"),
    ((gpu(6, 2, 16), gpu(6, 1, 16), gpu(6, 1, 16), STARTS), dict(frame=0), "frame"),
    ((gpu(6, 2, 16), gpu(6, 1, 16), gpu(6, 1, 16), STARTS), dict(frame=1.5), "frame"),
    ((gpu(6, 2, 16), gpu(6, 1, 16), gpu(6, 1, 16), STARTS), dict(scale=-1.0), "scale"),
    ((gpu(6, 2, 16).double(), gpu(6, 1, 16).double(), gpu(6, 1, 16).double(), STARTS), {}, "unsupported dtype"),
])
def test_python_checks(args, kw, message, monkeypatch):
    from d2conv3d_amd import attention
    monkeypatch.setattr(attention, "_try_native", lambda *a: None)
    with pytest.raises(RuntimeError, match=message):
        d2c.packed_attention(*args, **kw)


def test_cpu_tensors_are_refused():
    t = torch.zeros(6, 2, 16)
    with pytest.raises(RuntimeError, match="on the GPU"):
        d2c.packed_attention(t, t, t, torch.tensor([0, 6]))
    with pytest.raises(RuntimeError, match="must be a Tensor"):
        d2c.packed_attention(*(t.as_subclass(OnTheGpu),) * 3, [0, 6])
