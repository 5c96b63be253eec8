"""The memory's calls whose scores or ranks have no room at once, by what tables have room for: streams taken some at a time, the same results."""
import ctypes
import math

import pytest
import torch

import _memory
import d2conv3d_amd as d2c
from _memory import assert_same, make, on
from d2conv3d_amd import _lib

pytestmark = pytest.mark.gpu


def wide(lengths, page, heads, D, dtype, seed, slots):
    """A memory whose table has room for `slots` tokens of each stream, of which the pages behind what it has are not there."""
    m = make(lengths, page, heads, D, dtype, seed)
    table = torch.full((len(lengths), slots // page), -1, dtype=torch.int32)
    table[:, :m["table"].shape[1]] = m["table"]
    return dict(m, table=table)


def desc(m, heads):
    from d2conv3d_amd.memory import _memory_desc
    return _memory_desc("test", m), _lib.MemoryQueryDesc(heads, 0.1, (ctypes.c_int64 * 2)(heads * m.key.shape[3], m.key.shape[3]))


@pytest.mark.parametrize("dtype,hq,heads,streams", [(torch.bfloat16, 16, 4, 41), (torch.float32, 12, 1, 50), (torch.bfloat16, 24, 2, 23), (torch.bfloat16, 17, 1, 34)])
def test_tracked_attention(dtype, hq, heads, streams, dev):
    slots, D = 129600 // 16 * 16, 40
    lengths = [(i * 97) % 700 for i in range(streams)]
    m = wide(lengths, 16, heads, D, dtype, 1, slots)
    memory = on(dev, m)
    q, x = desc(memory, hq)
    assert streams * hq * slots * 4 > 256 << 20 > _lib.load().d2c_memory_attention_workspace_bytes(ctypes.byref(q), ctypes.byref(x), 1) - (16 << 20)
    print("memory_attention", dtype, hq, heads, streams, flush=True)
    query = torch.randn(streams, hq, D, generator=torch.Generator().manual_seed(2)).to(dtype)
    out, weights, bound, ubound = _memory.attend(m, query, 1.0 / math.sqrt(D))
    apart = torch.zeros(streams, 2, hq, D, dtype=dtype, device=dev)      # (streams of a projection)
    apart[:, 1] = query.to(dev)
    got = d2c.memory_attention(apart[:, 1], memory, track=True)
    assert bool(((got.cpu().double() - out).abs() <= bound).all())
    assert bool(((memory.usage.cpu().double() - (m["usage"].double() + weights)).abs() <= ubound).all())
    assert_same(memory, dict(m, usage=memory.usage.cpu()), "usage alone")
    assert torch.equal(d2c.memory_attention(query.to(dev), memory), d2c.memory_attention(apart[:, 1], memory))


def test_eviction(dev):
    lengths, slots = [(i * 31) % 90 for i in range(70)], 1 << 20
    m = wide(lengths, 64, 4, 8, torch.float32, 3, slots)
    memory = on(dev, m)
    assert 70 * 4 * slots * 4 > 1 << 30 > _lib.load().d2c_memory_evict_workspace_bytes(ctypes.byref(desc(memory, 4)[0]), 33)
    memory.evict(33, 5)
    assert_same(memory, _memory.evict(m, 33, 5))
