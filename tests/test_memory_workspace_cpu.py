"""Workspaces of the memory's calls go by what tables have room for, up to a limit: streams are then taken some at a time.  Without a GPU."""
import ctypes

import pytest

from d2conv3d_amd import _lib
from test_memory_cpu import asked, desc

MB = 1 << 20


def room(slots, **kw):
    return desc(page=64, per_stream=slots // 64, table_stride=slots // 64, **kw)


@pytest.mark.parametrize("streams", [1, 9, 10, 64, 1000])
@pytest.mark.parametrize("heads,query_heads", [(8, 8), (8, 48), (1, 32), (2, 128)])
@pytest.mark.parametrize("dtype", [0, 2])
def test_tracked_attention(streams, heads, query_heads, dtype):
    lib = _lib.load()

    def asks(track, slots, n=streams):
        return lib.d2c_memory_attention_workspace_bytes(ctypes.byref(room(slots, streams=n, heads=heads, dtype=dtype, pages=5000)), ctypes.byref(asked(query_heads)), track)
    slots = 129600 // 64 * 64
    one, plain = asks(1, slots, 1), asks(0, slots)
    assert 4 * query_heads * slots <= one
    assert 0 < asks(1, slots) <= max(256 * MB, one) + plain + 4096
    if streams * 4 * query_heads * slots <= 200 * MB:
        assert asks(1, slots) - plain >= streams * 4 * query_heads * slots


def test_eviction():
    lib = _lib.load()
    for streams in (1, 8, 64, 512, 5000):
        for slots, keep in ((129600 // 64 * 64, 60000), (1 << 20, 1000), (1 << 24, 1 << 23)):
            one = lib.d2c_memory_evict_workspace_bytes(ctypes.byref(room(slots, streams=1, heads=8)), keep)
            nb = lib.d2c_memory_evict_workspace_bytes(ctypes.byref(room(slots, streams=streams, heads=8)), keep)
            assert 8 * 4 * slots < one <= nb <= max(1024 * MB, one) + 65536
            if streams * one <= 1024 * MB:
                assert nb > streams * (one - 4096)
    # what is asked for is wanted
    q, some = room(1 << 20, streams=64, heads=8), ctypes.c_void_p(1 << 20)
    nb = lib.d2c_memory_evict_workspace_bytes(ctypes.byref(q), 1000)
    assert lib.d2c_memory_evict(ctypes.byref(q), *(some,) * 7, 1000, 0, some, nb - 1, None) != 0 and "workspace" in _lib.last_error()
    nb = lib.d2c_memory_attention_workspace_bytes(ctypes.byref(q), ctypes.byref(asked(48)), 1)
    assert lib.d2c_memory_attention(ctypes.byref(q), ctypes.byref(asked(48)), *(some,) * 7, some, nb - 1, None) != 0 and "workspace" in _lib.last_error()
