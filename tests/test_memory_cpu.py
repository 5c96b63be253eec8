"""What the memory in pages refuses, and what it asks for, without a GPU."""
import ctypes
import math

import pytest
import torch

import d2conv3d_amd as d2c
from d2conv3d_amd import _lib


def desc(**kw):
    base = dict(streams=2, heads=2, D=64, dtype=0, pages=8, page=16, per_stream=4, table_stride=4)
    base.update(kw)
    return _lib.MemoryDesc(*base.values(), (ctypes.c_int64 * 3)(2048, 1024, 64), (ctypes.c_int64 * 3)(2048, 1024, 64))


def asked(heads=4, scale=0.125):
    return _lib.MemoryQueryDesc(heads, scale, (ctypes.c_int64 * 2)(256, 64))


def attention(q, x):
    lib = _lib.load()
    return lib.d2c_memory_attention(ctypes.byref(q), ctypes.byref(x), *(None,) * 8, 0, None), _lib.last_error()


@pytest.mark.parametrize("change,message", [
    (dict(dtype=1), "float32 or bfloat16"), (dict(D=129), "128"), (dict(D=0), "positive"), (dict(heads=0), "positive"), (dict(page=0), "positive"),
    (dict(streams=-1), "negative"), (dict(pages=-1), "negative"), (dict(per_stream=-1), "negative"), (dict(per_stream=1 << 26), "too many"),
    (dict(streams=1 << 20), "too many"), (dict(streams=1 << 19, heads=4), "too many")])
def test_descriptions_that_are_refused(change, message):
    lib = _lib.load()
    q = desc(**change)
    rc, error = attention(q, asked())
    assert rc != 0 and message in error
    strides = (ctypes.c_int64 * 2)(128, 64)
    assert lib.d2c_memory_append(ctypes.byref(q), *(None,) * 9, strides, strides, None, 2, None) != 0 and message in _lib.last_error()
    assert lib.d2c_memory_evict(ctypes.byref(q), *(None,) * 7, 3, 0, None, 0, None) != 0 and message in _lib.last_error()
    assert lib.d2c_memory_attention_workspace_bytes(ctypes.byref(q), ctypes.byref(asked()), 1) == 0
    assert lib.d2c_memory_evict_workspace_bytes(ctypes.byref(q), 3) == 0


@pytest.mark.parametrize("heads,scale,message", [(3, 1.0, "multiple"), (0, 1.0, "multiple"), (-2, 1.0, "multiple"), (1024, 1.0, "256"), (4, 0.0, "scale"),
                                                 (4, -1.0, "scale"), (4, math.inf, "scale"), (4, math.nan, "scale")])
def test_queries_that_are_refused(heads, scale, message):
    rc, error = attention(desc(), asked(heads, scale))
    assert rc != 0 and message in error


def test_calls_that_are_refused():
    lib = _lib.load()
    rc, error = attention(desc(), asked())
    assert rc != 0 and "null" in error
    strides = (ctypes.c_int64 * 2)(128, 64)
    assert lib.d2c_memory_append(ctypes.byref(desc()), *(None,) * 9, strides, strides, None, 2, None) != 0 and "null" in _lib.last_error()
    for tokens in (-1, 3, 1 << 40):
        assert lib.d2c_memory_append(ctypes.byref(desc()), *(None,) * 9, strides, strides, None, tokens, None) != 0 and "tokens" in _lib.last_error()
    some = ctypes.c_void_p(4096)
    assert lib.d2c_memory_append(ctypes.byref(desc()), *(some,) * 9, None, strides, None, 2, None) != 0 and "null" in _lib.last_error()
    assert lib.d2c_memory_append(ctypes.byref(desc()), *(some,) * 9, strides, None, None, 2, None) != 0 and "null" in _lib.last_error()
    for keep, recent in ((0, 0), (-1, 0), (5, 6), (5, -1)):
        assert lib.d2c_memory_evict(ctypes.byref(desc()), *(None,) * 7, keep, recent, None, 0, None) != 0 and "keep" in _lib.last_error()
    # a workspace that is not there, too small, or not aligned
    nb = lib.d2c_memory_evict_workspace_bytes(ctypes.byref(desc()), 3)
    assert nb > 0
    for ws, have in ((None, 0), (ctypes.c_void_p(1 << 20), nb - 1), (ctypes.c_void_p((1 << 20) + 16), nb)):
        assert lib.d2c_memory_evict(ctypes.byref(desc()), *(some,) * 7, 3, 0, ws, have, None) != 0 and "workspace" in _lib.last_error()
        q = desc(per_stream=400, table_stride=400)
        assert lib.d2c_memory_attention(ctypes.byref(q), ctypes.byref(asked()), *(some,) * 7, ws, have, None) != 0 and "workspace" in _lib.last_error()


def test_nothing_to_do():
    lib = _lib.load()
    none = desc(streams=0)
    strides = (ctypes.c_int64 * 2)(128, 64)
    assert attention(none, asked())[0] == 0
    assert lib.d2c_memory_append(ctypes.byref(none), *(None,) * 9, strides, strides, None, 0, None) == 0
    assert lib.d2c_memory_evict(ctypes.byref(none), *(None,) * 7, 3, 0, None, 0, None) == 0
    assert lib.d2c_memory_evict(ctypes.byref(desc()), *(None,) * 7, 64, 0, None, 0, None) == 0      # (as many as there are slots)


def test_workspaces():
    lib = _lib.load()

    def asks(track, **kw):
        return lib.d2c_memory_attention_workspace_bytes(ctypes.byref(desc(**kw)), ctypes.byref(asked()), track)
    assert asks(0) == 0                                                       # short: one launch
    assert asks(1) == 2 * 4 * 64 * 4                                          # ... and the scores
    long = dict(per_stream=1000, table_stride=1000, pages=2000)
    assert asks(0, **long) > 0 and asks(1, **long) - asks(0, **long) == 2 * 4 * 16000 * 4
    assert lib.d2c_memory_evict_workspace_bytes(ctypes.byref(desc()), 64) == 0
    assert lib.d2c_memory_evict_workspace_bytes(ctypes.byref(desc()), 63) > 0


def test_python_refuses_what_is_not_on_the_gpu():
    memory = d2c.PagedMemory.empty(2, 40, 2, 16, device="cpu")
    assert memory.capacity == 64 and memory.table.tolist() == [[0], [1]] and memory.key.shape == (2, 2, 64, 16)
    q = torch.zeros(2, 4, 16, dtype=torch.bfloat16)
    for call in (lambda: memory.attend(q), lambda: memory.append(q[:, :2], q[:, :2]), lambda: memory.evict(3)):
        with pytest.raises(RuntimeError, match="on the GPU"):
            call()
    for call in (lambda: d2c.memory_attention(q, None), lambda: d2c.memory_append((), q, q), lambda: d2c.memory_evict(q, 3)):
        with pytest.raises(RuntimeError, match="PagedMemory"):
            call()
    for kw in (dict(streams=-1), dict(capacity=1.5), dict(heads=0), dict(channels=0), dict(page=0)):
        with pytest.raises(RuntimeError, match="whole number"):
            d2c.PagedMemory.empty(**{**dict(streams=1, capacity=1, heads=1, channels=1, device="cpu"), **kw})


class OnTheGpu(torch.Tensor):
    """A CPU tensor that says it is on the GPU: what the argument checks look at, with no memory touched."""
    is_cuda = True


@pytest.mark.parametrize("field,value,message", [
    ("key", lambda t: t[0], "must be"), ("key", lambda t: t.half(), "float32 or bfloat16"), ("value", lambda t: t[:, :1], "must be"), ("value", lambda t: t.float(), "both the same"),
    ("table", lambda t: t.long(), "table"), ("table", lambda t: t.t().contiguous().t(), "table"), ("lengths", lambda t: t[:1], "lengths"), ("lengths", lambda t: t.long(), "lengths"),
    ("seen", lambda t: t.float(), "seen"), ("usage", lambda t: t.double(), "usage"), ("usage", lambda t: t[:1], "usage"), ("positions", lambda t: t.float(), "positions"),
    ("positions", lambda t: t.transpose(1, 2), "positions")])
def test_memories_that_are_refused(field, value, message):
    from d2conv3d_amd.memory import _memory_desc
    memory = d2c.PagedMemory.empty(2, 40, 2, 16, page=8, device="cpu")
    for name in d2c.PagedMemory.__slots__:
        setattr(memory, name, getattr(memory, name).as_subclass(OnTheGpu))
    q = _memory_desc("x", memory)
    assert (q.streams, q.heads, q.D, q.pages, q.page, q.per_stream, list(q.key_stride)) == (2, 2, 16, 10, 8, 5, [256, 128, 16])
    setattr(memory, field, value(getattr(memory, field)))
    with pytest.raises(RuntimeError, match=message):
        _memory_desc("x", memory)
