"""The memory in pages on the GPU against plain loops: what is copied to the bit, outputs and weights against float64 within what
float32 arithmetic and one rounding of the result allow."""
import math

import pytest
import torch

import _memory
import d2conv3d_amd as d2c
from _memory import assert_same, make, on

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]

CASES = [
    # lengths, page, query heads, heads, channels
    ([1], 16, 1, 1, 64),
    ([0], 16, 2, 1, 32),
    ([7, 0, 1], 4, 4, 2, 40),
    ([350], 16, 8, 8, 32),
    ([65, 64, 63, 1], 64, 4, 1, 64),
    ([300, 17], 50, 6, 3, 24),
    ([129, 1000], 8, 8, 1, 128),
    ([1000, 3, 0, 700, 2000], 64, 16, 4, 64),
    ([900], 33, 3, 1, 7),
    ([700, 20], 1, 2, 2, 33),
    ([1500], 128, 12, 1, 96),           # more than eight rows of a key head
    ([100, 30], 16, 36, 2, 80),
    ([40], 16, 9, 1, 64),
    ([4000, 1], 64, 2, 1, 104),
    ([5000], 64, 5, 1, 127),
    ([3, 20], 8, 18, 1, 80),           # rows in groups, memories that one workgroup reads
    ([700, 0, 129], 64, 16, 2, 128),
    ([400, 1], 16, 16, 1, 32),
    ([256, 1000], 64, 34, 2, 64),
    ([31, 33], 16, 32, 1, 128),
    ([2000], 16, 33, 1, 40),
    ([5000, 40], 64, 70, 1, 88),
    ([100, 9000], 64, 6, 1, 20),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_attention(case, dtype, dev):
    print("memory_attention", case, dtype, flush=True)
    lengths, page, hq, heads, D = case
    m = make(lengths, page, heads, D, dtype, seed=sum(lengths) + D, per=max(-(-max(lengths) // page), 1) + 2)
    q = torch.randn(len(lengths), hq, D, generator=torch.Generator().manual_seed(D)).to(dtype)
    out, weights, bound, ubound = _memory.attend(m, q, 1.0 / math.sqrt(D))
    memory = on(dev, m)
    got = d2c.memory_attention(q.to(dev), memory)
    assert_same(memory, m, "read only")
    tracked = d2c.memory_attention(q.to(dev), memory, track=True)
    assert torch.equal(got, tracked)
    over = (got.cpu().double() - out).abs() / bound
    assert bool((over <= 1).all()), f"{over.max().item():.2f} of the bound"
    off = (memory.usage.cpu().double() - (m["usage"].double() + weights)).abs()
    assert bool((off <= ubound).all()), f"usage: {(off / ubound).max().item():.2f} of the bound"
    same = dict(m, usage=memory.usage.cpu())
    assert_same(memory, same, "usage alone")
    other = on(dev, m)
    assert torch.equal(d2c.memory_attention(q.to(dev), other, track=True), got) and torch.equal(other.usage, memory.usage)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_streams(dtype, dev):
    lengths = [(i * 37) % 90 if i % 5 else 0 for i in range(300)] + [3000]
    m = make(lengths, 16, 1, 32, dtype, seed=2)
    q = torch.randn(len(lengths), 4, 32, generator=torch.Generator().manual_seed(3)).to(dtype)
    out, weights, bound, ubound = _memory.attend(m, q, 0.3)
    memory = on(dev, m)
    got = memory.attend(q.to(dev), 0.3, True)
    assert bool(((got.cpu().double() - out).abs() <= bound).all())
    assert bool(((memory.usage.cpu().double() - m["usage"].double() - weights).abs() <= ubound).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1e-3, 30.0])
def test_scores_of_any_size(size, dtype, dev):
    m = make([600, 40], 16, 2, 64, dtype, seed=4)
    q = (torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(5)) * size).to(dtype)
    out, weights, bound, ubound = _memory.attend(m, q, 0.125)
    memory = on(dev, m)
    got = memory.attend(q.to(dev), track=True)
    assert bool(((got.cpu().double() - out).abs() <= bound).all())
    assert bool(((memory.usage.cpu().double() - m["usage"].double() - weights).abs() <= ubound).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("short", [True, False])
def test_pages_that_are_not_there(short, dtype, dev):
    """Numbers outside the pool, lengths outside the slots: slots that are not there, nothing else read or written."""
    lengths = [60, 90, 45, 30] if short else [600, 900, 450, 1]
    m = make(lengths, 16, 2, 40, dtype, seed=6)
    for place, number in (((0, 1), -1), ((1, 0), m["key"].shape[0]), ((1, 2), 2 ** 31 - 1), ((2, 0), -2 ** 31)):
        m["table"][place] = number
    m["lengths"][1], m["lengths"][3] = 2 ** 31 - 1, -7
    m["key"], m["value"] = (torch.nan_to_num(m[f], nan=0.5) for f in ("key", "value"))      # (stream 1 has every slot now)
    q = torch.randn(4, 2, 40, generator=torch.Generator().manual_seed(7)).to(dtype)
    out, weights, bound, ubound = _memory.attend(m, q, 0.2)
    memory = on(dev, m)
    got = memory.attend(q.to(dev), 0.2, True)
    assert bool(((got.cpu().double() - out).abs() <= bound).all())
    assert not bool(got[3].any())
    assert bool(((memory.usage.cpu().double() - m["usage"].double() - weights).abs() <= ubound).all())
    # a stream none of whose pages are there
    m["table"][0] = -1
    memory = on(dev, m)
    assert not bool(memory.attend(q.to(dev), 0.2, True)[0].any())
    new = [torch.randn(4, 2, 40, generator=torch.Generator().manual_seed(i)).to(dtype) for i in (8, 9)]
    m["usage"] = memory.usage.cpu()
    memory.append(*(t.to(dev) for t in new))
    m = _memory.append(m, *new)
    assert_same(memory, m, "append")
    memory.evict(20, 4)
    assert_same(memory, _memory.evict(m, 20, 4), "evict")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("length,hq", [(60, 1), (60, 4), (60, 8), (60, 20), (4000, 1), (4000, 4), (4000, 7), (4000, 16), (4000, 40)])
def test_infinities_that_are_read(length, hq, dtype, dev):
    """An infinite value, or one that is no number, in a slot that is there is all of its channel; a score of -infinity has no weight, one of
    +infinity leaves no number."""
    D, slot = 40, 37
    m = make([length, length], 16, 1, D, dtype, 71)
    q = torch.randn(2, hq, D, generator=torch.Generator().manual_seed(72)).to(dtype)
    q[:, :, 5] = torch.where(torch.arange(hq) % 2 == 0, -1.0, 1.0).to(dtype)
    at = (int(m["table"][1, slot // 16]), 0, slot % 16)
    as_it_is = on(dev, m).attend(q.to(dev)).cpu()
    for i, x in enumerate((math.inf, -math.inf, math.nan)):
        m["value"][at][i] = x
    here = on(dev, m).attend(q.to(dev)).cpu()
    assert torch.equal(here[0], as_it_is[0]) and torch.equal(here[1, :, 3:], as_it_is[1, :, 3:])
    assert bool((here[1, :, 0] == math.inf).all()) and bool((here[1, :, 1] == -math.inf).all()) and bool(here[1, :, 2].isnan().all())
    m["value"][at] = 1.0
    m["key"][at][5] = math.inf
    here = on(dev, m).attend(q.to(dev)).cpu()
    assert torch.equal(here[0], as_it_is[0]) and bool(here[1, 1::2].isnan().all())
    m["key"][at] = 0.0
    m["key"][at][5] = torch.finfo(dtype).max / 4      # (a finite score so low that its weight is 0 as well)
    low = on(dev, m).attend(q.to(dev)).cpu()
    assert torch.equal(here[1, 0::2], low[1, 0::2])


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype, dev):
    """Pages with the heads inside, a query that is part of a projection, rows of a table that lie apart, heads at an odd place."""
    m = make([200, 77], 16, 2, 40, dtype, seed=10, garbage=0.0)
    q = torch.randn(2, 4, 40, generator=torch.Generator().manual_seed(11)).to(dtype)
    out, _, bound, _ = _memory.attend(m, q, 0.15)
    memory = on(dev, m)
    want = memory.attend(q.to(dev), 0.15)
    assert bool(((want.cpu().double() - out).abs() <= bound).all())
    wide = torch.zeros(2, 3, 4, 43, dtype=dtype, device=dev)
    wide[:, 1, :, 1:41] = q.to(dev)
    pages = torch.full((*m["key"].shape[:1], 16, 2, 2, 41), math.nan, dtype=dtype, device=dev)
    for i, f in enumerate(("key", "value")):
        pages[:, :, i, :, 1:] = m[f].to(dev).transpose(1, 2)
    table = torch.full((2, 2, memory.table.shape[1]), -1, dtype=torch.int32, device=dev)
    table[:, 1] = memory.table
    apart = d2c.PagedMemory(*(pages[:, :, i, :, 1:].transpose(1, 2) for i in (0, 1)), table[:, 1], memory.lengths, memory.seen, memory.usage, memory.positions)
    assert torch.equal(apart.attend(wide[:, 1, :, 1:41], 0.15), want)
    new = torch.randn(2, 2, 2, 45, generator=torch.Generator().manual_seed(12)).to(dtype)
    m = _memory.append(m, new[:, 0, :, 5:], new[:, 1, :, 5:])
    assert memory.capacity > 200
    apart.append(*(new.to(dev)[:, i, :, 5:] for i in (0, 1)))
    for i, f in enumerate(("key", "value")):
        assert torch.equal(getattr(apart, f).cpu(), m[f])
    assert bool(pages[..., 0].isnan().all())
    apart.evict(90, 10)
    m = _memory.evict(m, 90, 10)
    for f in _memory.FIELDS:
        assert torch.equal(getattr(apart, f).cpu(), m[f]), f


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,page", [(64, 16), (40, 7), (7, 1), (128, 64)])
def test_append(D, page, dtype, dev):
    m = make([0, 3, 20, 16], page, 3, D, dtype, seed=13, per=-(-40 // page))
    gen = torch.Generator().manual_seed(14)
    memory = on(dev, m)
    for starts in ([0, 5, 5, 6, 30], None, [2, 3, 3, 9, 9], [0, 1, 40, 44, 45]):       # (the third stream runs out of slots)
        tokens = 4 if starts is None else 50
        k, v = (torch.randn(tokens, 3, D, generator=gen).to(dtype) for _ in range(2))
        m = _memory.append(m, k, v, starts)
        # (whole numbers of any width)
        first = None if starts is None else torch.tensor(starts, device=dev, dtype=torch.int64 if starts[0] else torch.int32)
        memory.append(k.to(dev), v.to(dev), first)
        assert_same(memory, m, str(starts))


def test_starts_that_do_not_rise(dev):
    """No token and no slot outside the tensors, whatever the starts are."""
    m = make([3, 4], 8, 1, 16, torch.float32, seed=15, per=4, garbage=0.0)
    k, v = (torch.randn(6, 1, 16, generator=torch.Generator().manual_seed(i)) for i in (16, 17))
    memory = on(dev, m)
    memory.append(k.to(dev), v.to(dev), torch.tensor([-5, 4, 100], device=dev, dtype=torch.int32))
    assert_same(memory, _memory.append(m, k, v, [0, 4, 6]))
    memory = on(dev, m)
    memory.append(k.to(dev), v.to(dev), torch.tensor([5, 2, 1], device=dev, dtype=torch.int32))
    torch.cuda.synchronize()
    assert memory.lengths.tolist() == [3, 4] and memory.seen.tolist() == m["seen"].tolist()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,page,heads,D,keep,recent", [
    ([40], 16, 1, 64, 39, 0), ([40], 16, 1, 64, 1, 1), ([40], 16, 2, 64, 20, 20), ([100, 20, 0, 64, 33], 16, 3, 40, 33, 5), ([200, 300], 50, 2, 24, 150, 149),
    ([2500, 64], 64, 2, 32, 1300, 200), ([4100], 128, 1, 128, 64, 0), ([1025, 1024, 1026], 8, 1, 7, 1024, 100),
    ([9000, 8192, 100], 64, 1, 8, 4000, 4000), ([20000], 50, 1, 8, 15000, 1), ([33000, 32769], 64, 1, 8, 20000, 3000), ([70001], 16, 1, 8, 66000, 100)])
def test_evict(lengths, page, heads, D, keep, recent, dtype, dev):
    m = make(lengths, page, heads, D, dtype, seed=keep)
    memory = on(dev, m)
    memory.evict(keep, recent)
    assert_same(memory, _memory.evict(m, keep, recent))


@pytest.mark.parametrize("usage", ["equal", "few", "zeros", "wild"])
def test_evict_ranks(usage, dev):
    """Ties go to the lower slot; zeros of either sign are one number; NaN is above, infinities at the ends."""
    m = make([700, 900], 32, 2, 16, torch.float32, seed=18)
    gen = torch.Generator().manual_seed(19)
    m["usage"] = {"equal": torch.full_like(m["usage"], 0.25), "few": torch.randint(0, 3, m["usage"].shape, generator=gen) / 4.0,
                  "zeros": torch.where(torch.rand(m["usage"].shape, generator=gen) < 0.5, 0.0, -0.0),
                  "wild": torch.tensor([math.nan, -math.nan, math.inf, -math.inf, -1.0, 0.0, 1e-42, 3.0])[torch.randint(0, 8, m["usage"].shape, generator=gen)]}[usage]
    memory = on(dev, m)
    memory.evict(411, 37)
    assert_same(memory, _memory.evict(m, 411, 37))


def test_evict_leaves_short_streams(dev):
    m = make([30, 12], 16, 2, 16, torch.bfloat16, seed=20)
    memory = on(dev, m)
    for keep in (30, 1000):
        memory.evict(keep, 3)
        assert_same(memory, m)


@pytest.mark.parametrize("dtype", DTYPES)
def test_captured_and_replayed(dtype, dev):
    """A stream's step in a graph: append, read with weights added up, evict.  Every replay is the step as it runs without one."""
    def fresh():
        m = make([30, 7, 64], 16, 2, 64, dtype, seed=21, per=6, garbage=0.0)
        return on(dev, m)
    gen = torch.Generator().manual_seed(22)
    tokens = [[torch.randn(3, h, 64, generator=gen).to(dtype).to(dev) for h in (2, 2, 4)] for _ in range(8)]
    eager, held = fresh(), fresh()
    static = [t.clone() for t in tokens[0]]

    def step(memory, k, v, q):
        memory.append(k, v)
        out = memory.attend(q, track=True)
        memory.evict(66, 20)
        return out
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(fresh(), *static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(held, *static)
    again = fresh()
    for f in _memory.FIELDS:
        getattr(held, f).copy_(getattr(again, f))
    for i, t in enumerate(tokens):
        want = step(eager, *t)
        for a, b in zip(static, t):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, want), i
        assert_same(held, {f: getattr(eager, f).cpu() for f in _memory.FIELDS}, str(i))
    assert eager.lengths.tolist() == [38, 15, 66] and eager.seen.tolist() == [43, 20, 77]


def test_another_stream(dev):
    m = make([500, 90], 16, 2, 64, torch.bfloat16, seed=23)
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(24)).to(torch.bfloat16).to(dev)
    want = on(dev, m).attend(q)
    memories = [on(dev, m) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for s, memory in zip(streams, memories):
            with torch.cuda.stream(s):
                outs.append(memory.attend(q, track=True))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs) and torch.equal(memories[0].usage, memories[1].usage)


def test_offsets_beyond_32_bits(dev):
    """Pages whose elements lie behind the 2^31st and, in bytes, the 2^32nd."""
    D, page = 128, 1024
    pages = 2 ** 31 // (D * page) + 40
    pool = torch.zeros((pages, 1, page, D), dtype=torch.bfloat16, device=dev)
    m = make([3000], page, 1, D, torch.bfloat16, seed=25)
    q = torch.randn(1, 2, D, generator=torch.Generator().manual_seed(26)).to(torch.bfloat16)
    near = on(dev, m)
    table = torch.tensor([[pages - 1, 5, pages - 20, 7]], dtype=torch.int32, device=dev)[:, :near.table.shape[1]].contiguous()
    pool[table[0].long()] = torch.nan_to_num(near.key[near.table[0].long()], nan=0.0)
    usage = torch.zeros((pages, 1, page), device=dev)
    usage[table[0].long()] = near.usage[near.table[0].long()]
    positions = torch.zeros((pages, 1, page), dtype=torch.int32, device=dev)
    positions[table[0].long()] = near.positions[near.table[0].long()]
    near.key = torch.nan_to_num(near.key, nan=0.0)
    near.value = near.key.clone()
    far = d2c.PagedMemory(pool, pool.clone(), table, near.lengths.clone(), near.seen.clone(), usage, positions)
    new = torch.randn(1, 1, D, generator=torch.Generator().manual_seed(27)).to(torch.bfloat16).to(dev)
    for memory in (near, far):
        memory.append(new, new)
    assert torch.equal(near.attend(q.to(dev), track=True), far.attend(q.to(dev), track=True))
    for memory in (near, far):
        memory.evict(1500, 10)
    for f in ("key", "value", "usage", "positions"):
        assert torch.equal(getattr(near, f)[near.table[0].long()], getattr(far, f)[table[0].long()]), f


def test_both_routes(dev, monkeypatch):
    """The Python functions and the native ones make the same calls; both say that they have changed what they change."""
    from d2conv3d_amd import _ops
    m = make([40, 90], 16, 2, 40, torch.float32, seed=28)
    gen = torch.Generator().manual_seed(29)
    q, k, v = (torch.randn(2, h, 40, generator=gen).to(dev) for h in (4, 2, 2))
    results = []
    for native in (True, False):
        if not native:
            monkeypatch.setattr(_ops, "_native", type("None_", (), {"__getattr__": lambda self, name: lambda *a: None})())
        memory = on(dev, m)
        versions = [getattr(memory, f)._version for f in _memory.FIELDS]
        memory.append(k, v)
        out = memory.attend(q, track=True)
        memory.evict(50, 5)
        after = [getattr(memory, f)._version for f in _memory.FIELDS]
        assert [a > b for a, b in zip(after, versions)] == [f != "table" for f in _memory.FIELDS]
        results.append([out, *(getattr(memory, f).nan_to_num(nan=-5.0) for f in _memory.FIELDS)])
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_no_streams_and_no_pages(dev):
    none = d2c.PagedMemory.empty(0, 10, 2, 16, device=dev)
    assert none.append(*(torch.zeros(0, 2, 16, device=dev, dtype=torch.bfloat16),) * 2).attend(torch.zeros(0, 4, 16, device=dev, dtype=torch.bfloat16)).shape == (0, 4, 16)
    none.evict(3)
    bare = d2c.PagedMemory.empty(2, 0, 2, 16, device=dev)
    t = torch.ones(2, 2, 16, device=dev, dtype=torch.bfloat16)
    bare.append(t, t)
    assert bare.lengths.tolist() == [0, 0] and bare.seen.tolist() == [1, 1]
    assert not bool(bare.attend(t, track=True).any())
    bare.evict(3)


def test_streams_of_a_pool_without_pages(dev):
    """Tables whose every number is outside the pool, which has no page: nothing is read, streams lose what is not there."""
    m = make([20, 3, 0], 8, 2, 16, torch.float32, 61)
    memory = on(dev, {f: t[:0] if f in ("key", "value", "usage", "positions") else t for f, t in m.items()})
    t = torch.ones(3, 2, 16, device=dev)
    assert not bool(memory.attend(t, track=True).any())
    memory.evict(5, 2)
    assert memory.lengths.tolist() == [5, 3, 0] and memory.seen.tolist() == m["seen"].tolist()
    memory.append(t, t)
    assert memory.lengths.tolist() == [6, 4, 1] and memory.seen.tolist() == (m["seen"] + 1).tolist()
    assert not bool(memory.attend(t, track=True).any())


def test_more_pages_and_heads_than_32_bits_count(dev):
    """Usage and positions behind the 2^31st: a page's number times the heads."""
    heads, pages = 1 << 20, 2060
    gen = torch.Generator(device=dev).manual_seed(62)
    usage = torch.rand((4, heads, 1), generator=gen, device=dev)
    positions = torch.arange(4, dtype=torch.int32, device=dev).view(4, 1, 1).expand(4, heads, 1).contiguous()
    key = torch.randn((4, heads, 1, 1), generator=gen, device=dev).to(torch.bfloat16)
    count = torch.full((1,), 4, dtype=torch.int32, device=dev)
    at = torch.tensor([[pages - 1, 1, pages - 2, 0]], dtype=torch.int32, device=dev)

    def spread(t):
        out = torch.zeros((pages, *t.shape[1:]), dtype=t.dtype, device=dev)
        out[at[0].long()] = t
        return out
    far = d2c.PagedMemory(spread(key), spread(-key), at, count.clone(), count.clone(), spread(usage), spread(positions))
    near = d2c.PagedMemory(key, -key, torch.arange(4, dtype=torch.int32, device=dev).view(1, 4), count.clone(), count.clone(), usage.clone(), positions.clone())
    for memory in (near, far):
        memory.evict(2, 1)
    assert far.lengths.tolist() == [2]
    a, b, c = usage[:3, :, 0]
    best = torch.where((a >= b) & (a >= c), 0, torch.where(b >= c, 1, 2))      # (beside the newest, 3)
    assert torch.equal(near.positions[:2, :, 0].sort(dim=0).values.long(), torch.stack([best, torch.full_like(best, 3)]))
    for f in ("key", "value", "usage", "positions"):
        assert torch.equal(getattr(near, f), getattr(far, f)[at[0].long()]), f


def test_refused_on_the_gpu(dev):
    memory = d2c.PagedMemory.empty(2, 40, 2, 16, page=8, dtype=torch.float32, device=dev)
    q = torch.zeros(2, 4, 16, device=dev)
    k = torch.zeros(2, 2, 16, device=dev)
    for call, message in ((lambda: memory.attend(q[:, :3]), "multiple"), (lambda: memory.attend(q[:1]), "must be"), (lambda: memory.attend(q.bfloat16()), "must be"),
                          (lambda: memory.attend(q, 0.0), "scale"), (lambda: memory.attend(q, math.nan), "scale"), (lambda: memory.attend(q.cpu()), "on the GPU"),
                          (lambda: memory.attend(q.clone().requires_grad_()), "no gradient"), (lambda: memory.append(k.clone().requires_grad_(), k), "no gradient"),
                          (lambda: memory.append(k[:1], k[:1]), "one token of each"), (lambda: memory.append(k, k[:1]), "values"),
                          (lambda: memory.append(k, k, torch.zeros(2, device=dev, dtype=torch.int32)), "whole numbers"),
                          (lambda: memory.append(k, k, torch.zeros(3, device=dev)), "whole numbers"), (lambda: memory.evict(0), "positive"),
                          (lambda: memory.evict(2.5), "whole number"), (lambda: memory.evict(3, 0.5), "whole number"), (lambda: memory.evict(3, 4), "recent"), (lambda: memory.evict(3, -1), "recent")):
        with pytest.raises(RuntimeError, match=message):
            call()
    assert not bool(memory.lengths.any())
    # keys that lie in one place, and keys whose gradient is wanted, are read, but not written to
    for change in (lambda t: t[:1].expand(t.shape), lambda t: t.clone().requires_grad_()):
        for which in ("key", "value"):
            other = d2c.PagedMemory(*(getattr(memory, f) for f in _memory.FIELDS))
            setattr(other, which, change(getattr(memory, which)))
            for call in (lambda: other.append(k, k), lambda: other.evict(3)):
                with pytest.raises(RuntimeError, match="overlap themselves|no gradient"):
                    call()
            with torch.no_grad():
                other.attend(q)
    assert not bool(memory.lengths.any())
