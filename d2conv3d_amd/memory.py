"""A memory of keys and values that grows with a stream, read by one new token at a time.  (No counterpart in the reference, which
computes clip after clip.)

    PagedMemory        keys and values of streams in pages, with each slot's accumulated weight and position
    memory_append      new tokens of the streams, one of each or whole clips
    memory_attention   one new token of each stream reads what its stream has
    memory_evict       streams that are too long lose the tokens that were read least

For inference: nothing here is differentiated or recorded (a call whose gradient or tangent is wanted, or that torch.jit.trace would
record, is refused).  float32 and bfloat16; weights, sums and usage are held in float32.
"""
import ctypes
import math

import torch
from torch.autograd import forward_ad

from . import _lib
from ._ops import _DT, _ptr, _stream, _try_native, _workspace
from .attention import _check, _check_tensors, _heads_contiguous

_TYPES = (torch.float32, torch.bfloat16)


class PagedMemory:
    """Keys and values of streams, in pages of a pool.

    `key`, `value` [pages, heads, page, channels] (any strides with the channels adjacent); `table` [streams, pages of a stream]
    int32: slot s of stream n is slot s % page of page table[n, s // page] (a number outside the pool: those slots are not there);
    `lengths` [streams] int32: slots that a stream has; `seen` [streams] int32: tokens it has had; `usage` [pages, heads, page]
    float32: the weights that a slot's token has got; `positions` [pages, heads, page] int32: which of the stream's tokens it is.
    The tensors are the caller's, and all that a call changes.  Streams that are written to (reading with `track` writes usage) share no
    page, and none has a page twice."""

    __slots__ = ("key", "value", "table", "lengths", "seen", "usage", "positions")

    def __init__(self, key, value, table, lengths, seen, usage, positions):
        self.key, self.value, self.table, self.lengths = key, value, table, lengths
        self.seen, self.usage, self.positions = seen, usage, positions

    @classmethod
    def empty(cls, streams, capacity, heads, channels, page=64, dtype=torch.bfloat16, device="cuda"):
        """Streams without tokens, with pages of their own for `capacity` tokens each."""
        for name, v, least in (("streams", streams, 0), ("capacity", capacity, 0), ("heads", heads, 1), ("channels", channels, 1), ("page", page, 1)):
            _check(int(v) == v and v >= least, f"PagedMemory: {name} must be a whole number of at least {least}, got {v}")
        per = -(-capacity // page)
        pages = streams * per
        both = torch.zeros((2, pages, heads, page, channels), dtype=dtype, device=device)
        counts = torch.zeros((2, streams), dtype=torch.int32, device=device)
        return cls(both[0], both[1], torch.arange(pages, dtype=torch.int32, device=device).view(streams, per), counts[0], counts[1],
                   torch.zeros((pages, heads, page), dtype=torch.float32, device=device),
                   torch.zeros((pages, heads, page), dtype=torch.int32, device=device))

    @property
    def capacity(self):
        """Slots that a stream can have."""
        return self.table.size(1) * self.key.size(2)

    def append(self, key, value, starts=None):
        memory_append(self, key, value, starts)
        return self

    def attend(self, query, scale=None, track=False):
        return memory_attention(query, self, scale, track)

    def evict(self, keep, recent=0):
        memory_evict(self, keep, recent)
        return self


def _memory_desc(what, m, written=False):
    """The description of a memory, its tensors checked; `written`: the call changes keys and values."""
    _check(isinstance(m, PagedMemory), f"{what}: memory must be a PagedMemory")
    _check_tensors(what, **{name: getattr(m, name) for name in PagedMemory.__slots__})
    k = m.key
    _check(k.dim() == 4 and k.shape == m.value.shape,
           f"{what}: key and value must be [pages, heads, page, channels], got {tuple(k.shape)} and {tuple(m.value.shape)}")
    _check(k.dtype in _TYPES and m.value.dtype == k.dtype, f"{what}: key and value must be float32 or bfloat16, both the same")
    pages, heads, page, channels = k.shape
    _check(heads > 0 and page > 0 and channels > 0, f"{what}: heads, slots of a page and channels must be positive, got {tuple(k.shape)}")
    _check(channels <= 128, f"{what}: heads of up to 128 channels, got {channels}")
    _check(all(t.stride(3) == 1 or channels == 1 for t in (k, m.value)), f"{what}: the channels of key and value must be adjacent")
    if written:
        _check(all(t.size(i) <= 1 or t.stride(i) > 0 for t in (k, m.value) for i in range(3)), f"{what}: key and value must not overlap themselves (expanded tensors)")
        _no_gradient(what, k, m.value)
    _check(m.table.dim() == 2 and m.table.dtype == torch.int32 and (m.table.stride(1) == 1 or m.table.size(1) <= 1),
           f"{what}: table must be int32 [streams, pages of a stream], rows without gaps")
    streams = m.table.size(0)
    for name in ("lengths", "seen"):
        t = getattr(m, name)
        _check(t.dtype == torch.int32 and tuple(t.shape) == (streams,) and t.is_contiguous(), f"{what}: {name} must be int32 [{streams}], contiguous")
    for name, dtype in (("usage", torch.float32), ("positions", torch.int32)):
        t = getattr(m, name)
        _check(t.dtype == dtype and t.shape == k.shape[:3] and t.is_contiguous(), f"{what}: {name} must be {dtype} {tuple(k.shape[:3])}, contiguous")
    strides = [(ctypes.c_int64 * 3)(t.stride(0), t.stride(1), t.stride(2)) for t in (k, m.value)]
    return _lib.MemoryDesc(streams, heads, channels, _DT[k.dtype], pages, page, m.table.size(1), m.table.stride(0), *strides)


def _not_recorded(what, memory, *tensors):
    """No trace, of which the library's call would be no part, and no tangent, which the result would lack."""
    _check(not torch.jit.is_tracing(), f"{what} is not recorded by torch.jit.trace: call it outside of what is traced")
    if isinstance(memory, PagedMemory):
        tensors += (memory.key, memory.value, memory.usage)
    _check(all(forward_ad.unpack_dual(t).tangent is None for t in tensors if isinstance(t, torch.Tensor)),
           f"{what} takes no forward-mode tangent")


def _no_gradient(what, *tensors):
    _check(not (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)), f"{what} takes no gradient: call it under torch.no_grad()")


def memory_append(memory, key, value, starts=None):
    """New tokens of the streams, behind those that are there: `key`, `value` [tokens, heads, channels] (any strides with the
    channels adjacent are read in place).  One token of each stream, in their order; or, with `starts` [streams + 1] (whole numbers,
    rising), tokens starts[n] .. starts[n + 1] - 1 of stream n.  They begin with a usage of 0; lengths and seen grow.  Tokens that no
    slot is left for, or whose page is not there, are dropped."""
    if isinstance(memory, PagedMemory):
        m = memory
        if _try_native("memory_append", m.key, m.value, m.table, m.lengths, m.seen, m.usage, m.positions, key, value, starts):
            return
    _not_recorded("memory_append", memory, key, value)
    desc = _memory_desc("memory_append", memory, True)
    _check_tensors("memory_append", memory=memory.key, key=key, value=value, starts=starts)
    for name, t in (("key", key), ("value", value)):
        _check(t.dim() == 3 and tuple(t.shape[1:]) == (desc.heads, desc.D) and t.dtype == memory.key.dtype,
               f"memory_append: {name} must be {memory.key.dtype} [tokens, {desc.heads}, {desc.D}], got {t.dtype} {tuple(t.shape)}")
    tokens = key.size(0)
    _check(value.size(0) == tokens, f"memory_append: {tokens} keys and {value.size(0)} values")
    if starts is None:
        _check(tokens == desc.streams, f"memory_append: without starts one token of each of {desc.streams} streams, got {tokens}")
    else:
        _check(tuple(starts.shape) == (desc.streams + 1,) and not starts.is_floating_point() and not starts.is_complex() and starts.dtype != torch.bool,
               f"memory_append: starts must be {desc.streams + 1} whole numbers")
        starts = (starts.clamp(0, tokens) if starts.dtype == torch.int64 else starts).to(torch.int32).contiguous()
    _no_gradient("memory_append", key, value)
    key, value = (_heads_contiguous(t.detach()) for t in (key, value))
    ks, vs = ((ctypes.c_int64 * 2)(t.stride(0), t.stride(1)) for t in (key, value))
    changed = (memory.key, memory.value, memory.lengths, memory.seen, memory.usage, memory.positions)
    torch.autograd.graph.increment_version(changed)
    dev = memory.key.device
    with torch.cuda.device(dev):
        rc = _lib.load().d2c_memory_append(ctypes.byref(desc), _ptr(memory.key), _ptr(memory.value), _ptr(memory.table), _ptr(memory.lengths),
                                           _ptr(memory.seen), _ptr(memory.usage), _ptr(memory.positions), _ptr(key), _ptr(value), ks, vs,
                                           _ptr(starts), tokens, _stream(dev))
    _lib.check(rc, "memory_append")


def memory_attention(query, memory, scale=None, track=False):
    """softmax(scale * query key^T) value over the slots that each stream has: `query` [streams, query heads, channels] (any strides
    with the channels adjacent), one token of each stream, query heads a multiple of the memory's (h * query heads / heads .. share
    key head h, 256 at most); `scale` 1 / sqrt(channels) by default.  A stream without slots reads zeros; slots that are not there
    have no influence whatever they hold.  The work is split over the slots, evenly whatever the streams' lengths.

    `track`: the weights of the query heads that share a key head are added to the slots' usage, which memory_evict goes by."""
    if isinstance(memory, PagedMemory):
        m = memory
        out = _try_native("memory_attention", query, m.key, m.value, m.table, m.lengths, m.usage, m.positions, scale, bool(track))
        if out is not None:
            return out
    _not_recorded("memory_attention", memory, query)
    desc = _memory_desc("memory_attention", memory)
    _check_tensors("memory_attention", memory=memory.key, query=query)
    _check(query.dim() == 3 and query.size(0) == desc.streams and query.size(2) == desc.D and query.dtype == memory.key.dtype,
           f"memory_attention: query must be {memory.key.dtype} [{desc.streams}, heads, {desc.D}], got {query.dtype} {tuple(query.shape)}")
    heads = query.size(1)
    _check(heads > 0 and heads % desc.heads == 0, f"memory_attention: {heads} query heads are no positive multiple of {desc.heads} key heads")
    _check(heads // desc.heads <= 256, f"memory_attention: up to 256 query heads to a key head, got {heads // desc.heads}")
    scale = 1.0 / math.sqrt(desc.D) if scale is None else float(scale)
    _check(0.0 < scale < math.inf, f"memory_attention: scale must be positive and finite, got {scale}")
    _no_gradient("memory_attention", query, memory.key, memory.value)
    query = _heads_contiguous(query.detach())
    request = _lib.MemoryQueryDesc(heads, scale, (ctypes.c_int64 * 2)(query.stride(0), query.stride(1)))
    out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    if track:
        torch.autograd.graph.increment_version(memory.usage)
    lib, dev = _lib.load(), query.device
    with torch.cuda.device(dev):
        nb = lib.d2c_memory_attention_workspace_bytes(ctypes.byref(desc), ctypes.byref(request), int(bool(track)))
        ws = _workspace(nb, dev)
        rc = lib.d2c_memory_attention(ctypes.byref(desc), ctypes.byref(request), _ptr(query), _ptr(memory.key), _ptr(memory.value),
                                      _ptr(memory.table), _ptr(memory.lengths), _ptr(memory.usage if track else None), _ptr(out), _ptr(ws), nb,
                                      _stream(dev))
    _lib.check(rc, "memory_attention")
    return out


def memory_evict(memory, keep, recent=0):
    """Streams of more than `keep` tokens lose some, each head its own: the newest `recent` stay, and of the others those of the
    largest usage (the lower slot of two with the same; a usage that is no number counts as the largest), `keep` in all.  Tokens that
    stay behind slot keep - 1 move into the places of those that go, in order, with their usage and position; no other token moves.
    lengths becomes keep there.  Slots that are not there (of pages outside the pool) count and are the first to go; where one lies
    before `keep`, the token that would move into it is lost, even a newest one: let the pages of a stream's first `keep` slots be there."""
    for name, v in (("keep", keep), ("recent", recent)):
        _check(int(v) == v, f"memory_evict: {name} must be a whole number, got {v}")
    keep, recent = int(keep), int(recent)
    if isinstance(memory, PagedMemory):
        m = memory
        if _try_native("memory_evict", m.key, m.value, m.table, m.lengths, m.seen, m.usage, m.positions, keep, recent):
            return
    _not_recorded("memory_evict", memory)
    desc = _memory_desc("memory_evict", memory, True)
    _check(0 < keep < 1 << 31, f"memory_evict: keep must be positive, got {keep}")
    _check(0 <= recent <= keep, f"memory_evict: recent must be in 0 .. keep ({keep}), got {recent}")
    changed = (memory.key, memory.value, memory.lengths, memory.usage, memory.positions)
    torch.autograd.graph.increment_version(changed)
    lib, dev = _lib.load(), memory.key.device
    with torch.cuda.device(dev):
        nb = lib.d2c_memory_evict_workspace_bytes(ctypes.byref(desc), keep)
        ws = _workspace(nb, dev)
        rc = lib.d2c_memory_evict(ctypes.byref(desc), _ptr(memory.key), _ptr(memory.value), _ptr(memory.table), _ptr(memory.lengths),
                                  _ptr(memory.seen), _ptr(memory.usage), _ptr(memory.positions), keep, recent, _ptr(ws), nb, _stream(dev))
    _lib.check(rc, "memory_evict")
