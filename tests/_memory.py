"""A memory in pages restated in plain loops, in 64 bits on the CPU, and its inputs."""
import math

import torch

import d2conv3d_amd as d2c

U32, U16 = 2.0 ** -24, 2.0 ** -8
FIELDS = ("key", "value", "table", "lengths", "seen", "usage", "positions")


def make(lengths, page, heads, D, dtype, seed=0, per=None, garbage=math.nan):
    """A memory on the CPU: pages in any order, `garbage` in the slots that are not there (usage and positions, too)."""
    gen = torch.Generator().manual_seed(seed)
    n = len(lengths)
    per = max(-(-max([0, *lengths]) // page), 1) if per is None else per
    pages = n * per + 1                                  # (one page is nobody's)
    m = {"key": torch.randn(pages, heads, page, D, generator=gen).to(dtype), "value": torch.randn(pages, heads, page, D, generator=gen).to(dtype),
         "table": (torch.randperm(pages, generator=gen)[:n * per]).int().view(n, per), "lengths": torch.tensor(lengths, dtype=torch.int32),
         "seen": torch.tensor([max(length, 0) + 5 for length in lengths], dtype=torch.int32),
         "usage": torch.rand(pages, heads, page, generator=gen) ** 4, "positions": torch.zeros(pages, heads, page, dtype=torch.int32)}
    there = torch.zeros(pages, heads, page, dtype=torch.bool)
    for i, length in enumerate(lengths):
        length = min(max(length, 0), per * page)
        slot = torch.arange(length)
        at = m["table"][i].long()[slot // page], slice(None), slot % page
        m["positions"][at] = torch.stack([(torch.randperm(length, generator=gen) + 5).int() for _ in range(heads)], 1)
        there[at] = True
    m["key"][~there], m["value"][~there] = garbage, garbage
    m["usage"][~there], m["positions"][~there] = 1e30, 2 ** 31 - 1
    return m


def on(dev, m):
    return d2c.PagedMemory(*(m[f].to(dev) for f in FIELDS))


def slots_of(m, n):
    """(page, place) of the slots of a stream that are there, None for those whose page is not"""
    page, pages = m["key"].shape[2], m["key"].shape[0]
    length = min(max(int(m["lengths"][n]), 0), m["table"].shape[1] * page)
    return [(int(m["table"][n, s // page]), s % page) if 0 <= int(m["table"][n, s // page]) < pages else None for s in range(length)]


def attend(m, q, scale):
    """(out, weights added to usage) in float64, the bounds of both's errors."""
    n, hq, D = q.shape
    heads = m["key"].shape[1]
    group = hq // heads
    out, bound = torch.zeros(n, hq, D, dtype=torch.float64), torch.zeros(n, hq, D, dtype=torch.float64)
    usage, ubound = torch.zeros(m["usage"].shape, dtype=torch.float64), torch.zeros(m["usage"].shape, dtype=torch.float64)
    u = U16 if q.dtype == torch.bfloat16 else 0.0
    for i in range(n):
        at = [x for x in slots_of(m, i) if x is not None]
        if not at:
            continue
        page, place = (torch.tensor(t) for t in zip(*at))
        for h in range(hq):
            k, v = (m[name][page, h // group, place].double() for name in ("key", "value"))
            x = q[i, h].double()
            s = k @ x * scale
            # float32 products and sums over D channels, an exponential whose argument is rounded, sums over the slots
            e = U32 * (D + 64 + len(at) / 8 + 4 * ((k.abs() @ x.abs()) * scale).max())
            p = torch.softmax(s, 0)
            out[i, h] = p @ v
            bound[i, h] = 2 * e * (p @ v.abs()) + u * out[i, h].abs()
            usage[page, h // group, place] += p
            ubound[page, h // group, place] += (2 * e + group * U32) * p
    return out, usage, bound + 1e-30, ubound + 2 * U32 * m["usage"].double().abs()


def append(m, key, value, starts=None):
    """The memory after it."""
    m = {f: t.clone() for f, t in m.items()}
    page, pages = m["key"].shape[2], m["key"].shape[0]
    slots = m["table"].shape[1] * page
    for n in range(m["table"].shape[0]):
        t0, t1 = (n, n + 1) if starts is None else (min(max(int(s), 0), key.shape[0]) for s in starts[n:n + 2])
        length = min(max(int(m["lengths"][n]), 0), slots)
        for i in range(max(t1 - t0, 0)):
            s = length + i
            if s >= slots or not 0 <= int(m["table"][n, s // page]) < pages:
                continue
            at = int(m["table"][n, s // page]), slice(None), s % page
            m["key"][at], m["value"][at] = key[t0 + i], value[t0 + i]
            m["usage"][at], m["positions"][at] = 0.0, int(m["seen"][n]) + i
        m["lengths"][n] = min(length + max(t1 - t0, 0), slots)
        m["seen"][n] += max(t1 - t0, 0)
    return m


def evict(m, keep, recent):
    """The memory after it."""
    old, m = m, {f: t.clone() for f, t in m.items()}
    for n in range(m["table"].shape[0]):
        at = slots_of(old, n)
        if len(at) <= keep:
            continue
        m["lengths"][n] = keep
        for h in range(m["key"].shape[1]):
            page, place = (torch.tensor([0 if x is None else x[i] for x in at]) for i in (0, 1))
            usage, newest = old["usage"][page, h, place].tolist(), (old["positions"][page, h, place] >= int(old["seen"][n]) - recent).tolist()

            def rank(s):      # sorts as what stays first does
                if at[s] is None:
                    return (3, 0.0, s)
                if newest[s]:
                    return (0, 0.0, s)
                return (1, 0.0, s) if math.isnan(usage[s]) else (2, -usage[s], s)
            stays = set(sorted(range(len(at)), key=rank)[:keep])
            holes = [s for s in range(keep) if s not in stays]
            fillers = [s for s in range(keep, len(at)) if s in stays]
            assert len(holes) == len(fillers)
            for to, of in zip(holes, fillers):
                if at[to] is None or at[of] is None:
                    continue
                for f in ("key", "value", "usage", "positions"):
                    m[f][at[to][0], h, at[to][1]] = old[f][at[of][0], h, at[of][1]]
    return m


def assert_same(memory, m, what=""):
    """The same to the bit."""
    for f in FIELDS:
        a, b = getattr(memory, f).cpu(), m[f]
        assert a.dtype == b.dtype and a.shape == b.shape, (what, f)
        kind = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[a.element_size()]
        off = a.contiguous().view(kind) != b.contiguous().view(kind)
        assert not bool(off.any()), f"{what}: {f} differs at {int(off.sum())} places, first {off.nonzero()[0].tolist()}"
