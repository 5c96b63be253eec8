"""What is timed of the operators that read a clip token by token: causal attention over packed sequences (how such a network
is trained, and how it takes in a clip that is there from the start), the memory of keys and values in pages that grows with a
stream, its reading by one new token, and its eviction by the weight that its tokens have got.

A case is a dict of plain values:

  op        "packed" | "append" | "attend" | "evict"
  dtype     "f32" | "bf16": element type of queries, keys, values, outputs and gradients
  n         sequences (streams)
  longest   tokens of the longest sequence; the others have between none and that many (`spread` 0: all have as many)
  heads, kv_heads, d
  train     packed: forward and all gradients; otherwise forward only
  past      packed: how many keys a sequence may have in front of its queries (a clip that goes on), each its own number
  frame     packed: tokens of a frame, which read each other; 1: token after token
  page      slots of a page (memory)
  new       append: tokens of the longest piece that is appended; 1: one token of every stream
  track     attend: the weights are added up in the memory
  keep, recent   evict: tokens of a stream that stay, and how many of these are the newest whatever their weight
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- cases
def _packed(n, longest, heads, kv_heads, d, dtype, train, frame=1, past=0, spread=1.0):
    return dict(op="packed", n=n, longest=longest, heads=heads, kv_heads=kv_heads, d=d, dtype=dtype, train=train,
                frame=frame, past=past, spread=spread)


def _append(n, longest, new, kv_heads, d, dtype, page, spread=1.0):
    return dict(op="append", n=n, longest=longest, new=new, kv_heads=kv_heads, d=d, dtype=dtype, page=page, spread=spread)


def _attend(n, longest, heads, kv_heads, d, dtype, page, track=False, spread=1.0):
    return dict(op="attend", n=n, longest=longest, heads=heads, kv_heads=kv_heads, d=d, dtype=dtype, page=page,
                track=track, spread=spread)


def _evict(n, longest, keep, recent, kv_heads, d, dtype, page, spread=1.0):
    return dict(op="evict", n=n, longest=longest, keep=keep, recent=recent, kv_heads=kv_heads, d=d, dtype=dtype,
                page=page, spread=spread)


def listed():
    cases = {
        # a few small frames in inference: launches and host work count
        "packed small f32 infer": _packed(4, 350, 4, 4, 32, "f32", False),
        # odd sizes in float32, a training step
        "packed odd f32 train": _packed(3, 1417, 6, 3, 40, "f32", True),
        # clips of up to eight frames, the cells of a frame read each other: a training step
        "packed clips bf16 train": _packed(6, 12960, 8, 8, 64, "bf16", True, frame=1620),
        # pieces of clips that go on where earlier pieces ended
        "packed pieces bf16 infer": _packed(16, 4096, 16, 4, 128, "bf16", False, past=8192),
        # one long clip, token after token, keys shared by four heads each
        "packed long bf16 train": _packed(1, 25920, 8, 2, 64, "bf16", True, spread=0.0),
        # serving: one new token of each stream
        "append tokens bf16": _append(64, 4096, 1, 4, 64, "bf16", 64),
        # clips that are there from the start
        "append clips bf16": _append(4, 1620, 12960, 8, 64, "bf16", 64),
        # one stream that has just begun
        "attend short f32": _attend(1, 350, 8, 8, 32, "f32", 16),
        # many streams of their own lengths whose memories are to be evicted from later
        "attend streams bf16 track": _attend(32, 12960, 16, 4, 64, "bf16", 64, True),
        # two streams with very long memories
        "attend long bf16": _attend(2, 129600, 8, 2, 128, "bf16", 64, spread=0.0),
        # one stream, half of its memory goes; heads that are no power of two, small pages
        "evict small f32": _evict(1, 3240, 1620, 350, 4, 40, "f32", 16, spread=0.0),
        # streams of their own lengths, those that are too long lose what is read least
        "evict streams bf16": _evict(8, 25920, 12960, 1620, 8, 64, "bf16", 64, spread=0.5),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    largest = {}
    for c in listed():
        largest[c["op"]] = max(largest.get(c["op"], 0.0), _weight(c))
    while True:
        op = rng.choice(["packed", "packed", "attend", "attend", "evict", "append"])
        dtype = rng.choice(["f32", "bf16", "bf16"])
        kv = rng.choice([1, 2, 3, 4, 8])
        d = rng.choice([24, 32, 40, 64, 64, 80, 96, 128, 128])
        spread = rng.choice([0.0, 0.5, 1.0])
        page = rng.choice([8, 16, 16, 50, 64, 64, 128])
        if op == "packed":
            case = _packed(rng.choice([1, 1, 2, 3, 5, 16]), _log_int(rng, 1, 25920), kv * rng.choice([1, 1, 2, 4]), kv, d, dtype,
                           rng.random() < 0.6, rng.choice([1, 1, 1, 7, 350, 1620]), rng.choice([0, 0, _log_int(rng, 1, 12960)]), spread)
        elif op == "append":
            case = _append(_log_int(rng, 1, 64), _log_int(rng, 1, 12960), rng.choice([1, _log_int(rng, 2, 12960)]), kv, d, dtype,
                           page, spread)
        elif op == "attend":
            case = _attend(_log_int(rng, 1, 64), _log_int(rng, 1, 129600), kv * rng.choice([1, 2, 4, 8, 12]), kv, d, dtype, page,
                           rng.random() < 0.5, spread)
        else:
            longest = _log_int(rng, 16, 64800)
            keep = max(1, round(longest * rng.uniform(0.1, 0.95)))
            case = _evict(_log_int(rng, 1, 16), longest, keep, round(keep * rng.choice([0.0, 0.1, 0.5])), kv, d, dtype, page, spread)
        if _weight(case) <= largest[op]:
            return case


def _lengths(c, most, least=0, salt=0):
    """Lengths of the sequences: a part of the case, the same for every seed."""
    rng = random.Random(c["n"] * 1000003 + c["longest"] * 31 + salt)
    rest = [max(least, round(most * (1.0 - c["spread"] * rng.random()))) for _ in range(c["n"] - 1)]
    return [most] + rest


def _query_key_lengths(c):
    q = _lengths(c, c["longest"])
    past = _lengths(c, c["past"], 0, 1) if c["past"] else [0] * c["n"]
    return q, [a + b for a, b in zip(q, past)]


def _new_lengths(c):
    return [1] * c["n"] if c["new"] == 1 else _lengths(c, c["new"], 0, 2)


def _pairs_of(lq, lk, frame):
    """Keys that a sequence's queries read, all together."""
    return sum(min(lk, ((lk - lq + i) // frame + 1) * frame) for i in range(lq)) if frame > 1 else lq * (lk - lq) + lq * (lq + 1) // 2


def work(case):
    c, size = case, 2 if case["dtype"] == "bf16" else 4
    if c["op"] == "packed":
        lq, lk = _query_key_lengths(c)
        q, kv = sum(lq) * c["heads"] * c["d"], 2 * sum(lk) * c["kv_heads"] * c["d"]
        pairs = sum(_pairs_of(a, b, c["frame"]) for a, b in zip(lq, lk))
        return {"bytes": float((4 * q + 2 * kv if c["train"] else 2 * q + kv) * size),
                "flops": 4.0 * pairs * c["heads"] * c["d"] * (3.5 if c["train"] else 1)}
    row = 2 * c["d"] * size
    if c["op"] == "append":
        new = sum(_new_lengths(c)) * c["kv_heads"]
        return {"bytes": float(new * (2 * row + 8) + 16 * c["n"]), "flops": float(new * 2)}
    slots = sum(_lengths(c, c["longest"])) * c["kv_heads"]
    if c["op"] == "attend":
        return {"bytes": float(slots * (row + (8 if c["track"] else 0)) + 2 * c["n"] * c["heads"] * c["d"] * size),
                "flops": 4.0 * slots * c["heads"] // c["kv_heads"] * c["d"]}
    # tokens dropped among the first `keep`, whose places are taken by others
    moved = sum(c["keep"] * (1.0 - c["keep"] / n) for n in _lengths(c, c["longest"]) if n > c["keep"]) * c["kv_heads"]
    return {"bytes": 8.0 * slots + 2.0 * moved * (row + 8), "flops": float(slots)}


def _weight(c):
    """How much a case costs, roughly (a float32 product counts like six)."""
    w = work(c)
    return w["bytes"] + (w["flops"] * (6 if c["dtype"] == "f32" else 1) / 100 if c["op"] == "packed" else 0)


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    c, dev, dtype = case, torch.device("cuda"), DTYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(int(seed))

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * std).to(dtype)

    def starts(lengths):
        return torch.tensor([0] + lengths, device=dev).cumsum(0).int()

    state = {"case": c}
    if c["op"] == "packed":
        lq, lk = _query_key_lengths(c)
        inputs = [normal(sum(lq), c["heads"], c["d"]), normal(sum(lk), c["kv_heads"], c["d"]), normal(sum(lk), c["kv_heads"], c["d"])]
        state |= {"lengths": (lq, lk), "starts": starts(lq), "key_starts": starts(lk) if c["past"] else None,
                  "inputs": [t.requires_grad_(c["train"]) for t in inputs]}
        if c["train"]:
            state["grad_out"] = normal(*inputs[0].shape)
        return state

    # a memory in pages that streams have taken in any order
    have = _lengths(c, c["longest"])
    most = max(h + (m if c["op"] == "append" else 0) for h, m in zip(have, _new_lengths(c) if c["op"] == "append" else have))
    per = -(-most // c["page"])
    pages, kv, d = c["n"] * per, c["kv_heads"], c["d"]
    state["table"] = torch.randperm(pages, generator=gen, device=dev).int().view(c["n"], per)
    state["key"] = normal(pages, kv, c["page"], d)
    state["value"] = normal(pages, kv, c["page"], d)
    # lengths, tokens seen; weights added up and positions of the slots: two planes of one tensor each
    lengths = torch.tensor(have, device=dev).int()
    state["counts"] = torch.stack([lengths, lengths + 100])
    tokens = torch.empty(2, pages, kv, c["page"], dtype=torch.int32, device=dev)
    # a few tokens are read much, most of them little
    tokens[0] = torch.exp(torch.randn(pages, kv, c["page"], generator=gen, device=dev) * 2 - 3).view(torch.int32)
    # tokens lie in the order in which they came, but for those that have moved into others' places
    slot = torch.arange(per * c["page"], device=dev)
    key = slot + torch.rand(c["n"], kv, per * c["page"], generator=gen, device=dev) * (0.3 * c["longest"])
    key = torch.where(slot < lengths[:, None, None], key, 1e9)
    order = key.argsort(-1).argsort(-1).int() + 100
    tokens[1][state["table"].long().flatten()] = order.view(c["n"], kv, per, c["page"]).permute(0, 2, 1, 3).reshape(pages, kv, c["page"])
    state["tokens"] = tokens
    state["first"] = (state["counts"].clone(), tokens.clone())
    if c["op"] == "append":
        new = _new_lengths(c)
        state["starts"] = None if c["new"] == 1 else starts(new)
        # keys and values as one projection leaves them
        both = normal(sum(new), 2, kv, d)
        state["inputs"] = [both[:, 0], both[:, 1]]
    elif c["op"] == "attend":
        state["inputs"] = [normal(c["n"], c["heads"], d)]
    return state


# ---------------------------------------------------------------- the operators
def run(state):
    c = state["case"]
    if c["op"] == "packed":
        if not own:
            with torch.no_grad():
                return _plain_packed(state)
        if not c["train"]:
            with torch.no_grad():
                return _call_packed(state)
        out = _call_packed(state)
        return [out.detach(), *torch.autograd.grad(out, state["inputs"], state["grad_out"])]
    with torch.no_grad():
        # the memory as it was, so that every pass has the same to do
        if c["op"] != "attend":
            state["counts"].copy_(state["first"][0])
        if c["op"] == "evict" or c["op"] == "attend" and c["track"]:
            state["tokens"].copy_(state["first"][1])
        if own:
            return _call_memory(state)
        return {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict}[c["op"]](state)


def _call_packed(state):
    import d2conv3d_amd as d2c
    return d2c.packed_attention(*state["inputs"], state["starts"], state["key_starts"], causal=True, frame=state["case"]["frame"])


def _call_memory(state):
    import d2conv3d_amd as d2c
    c = state["case"]
    if "memory" not in state:      # (the handle that a program keeps of its memory)
        state["memory"] = d2c.PagedMemory(state["key"], state["value"], state["table"], state["counts"][0], state["counts"][1],
                                          state["tokens"][0].view(torch.float32), state["tokens"][1])
    memory = state["memory"]
    if c["op"] == "append":
        d2c.memory_append(memory, *state["inputs"], starts=state["starts"])
        return _memory_outputs(state)
    if c["op"] == "attend":
        out = d2c.memory_attention(state["inputs"][0], memory, track=c["track"])
        return [out, memory.usage] if c["track"] else out
    d2c.memory_evict(memory, c["keep"], c["recent"])
    return _memory_outputs(state)


def _memory_outputs(state):
    return {"key": state["key"], "value": state["value"], "lengths": state["counts"][0], "seen": state["counts"][1],
            "usage": state["tokens"][0].view(torch.float32), "positions": state["tokens"][1]}


# ... in elementary operations
def _plain_packed(state):
    """Sequences side by side, as long as the longest, where that is little; else one after the other."""
    c, (q, k, v) = state["case"], state["inputs"]
    lq, lk = state["lengths"]
    together = c["n"] * max(lq) * max(lk) * c["heads"] <= 1 << 26
    groups = [(slice(0, sum(lq)), slice(0, sum(lk)), max(lq), max(lk), slice(0, c["n"] + 1))] if together else []
    q0 = k0 = 0
    for i, (a, b) in enumerate(zip(lq, lk) if not together else ()):
        groups.append((slice(q0, q0 + a), slice(k0, k0 + b), a, b, slice(i, i + 2)))
        q0, k0 = q0 + a, k0 + b
    outs = [torch.empty_like(q)] + ([torch.empty_like(t) for t in (q, k, v)] if c["train"] else [])
    for rows, keys, a, b, some in groups:
        if a == 0:
            for t in outs[2:]:
                t[keys] = 0
            continue
        parts = [q[rows], k[keys], v[keys]] + ([state["grad_out"][rows]] if c["train"] else [])
        starts = state["starts"][some]
        key_starts = starts if state["key_starts"] is None else state["key_starts"][some]
        results = _plain_sequences(parts, starts - starts[0], key_starts - key_starts[0], a, b, c["frame"])
        for t, at, r in zip(outs, (rows, rows, keys, keys), results):
            t[at] = r
    return outs if c["train"] else outs[0]


def _plain_sequences(parts, starts, key_starts, lq, lk, frame):
    """Sequences of up to lq queries and lk keys: [L, H, D] each, all behind each other; their output and gradients."""
    starts, key_starts = starts.long(), key_starts.long()
    dev, n, kv = parts[0].device, starts.shape[0] - 1, parts[1].shape[1]
    group, scale = parts[0].shape[1] // kv, 1.0 / math.sqrt(parts[0].shape[2])

    def by_head(x, starts, longest):     # [L, kv * s, D] -> [n * kv, s * longest, D]
        at = starts[:-1, None] + torch.arange(longest, device=dev)
        y = torch.where((at < starts[1:, None])[..., None, None], x[at.clamp(max=x.shape[0] - 1)].float(), 0.0)
        s = x.shape[1] // kv
        return y.view(n, longest, kv, s, -1).permute(0, 2, 3, 1, 4).reshape(n * kv, s * longest, -1)

    def back(x, starts, longest, like):  # ... and back
        s = like.shape[1] // kv
        token = torch.arange(like.shape[0], device=dev)
        which = torch.searchsorted(starts, token, right=True) - 1
        return x.view(n, kv, s, longest, -1).permute(0, 3, 1, 2, 4)[which, token - starts[which]].flatten(1, 2)

    q, g = (by_head(t, starts, lq) for t in (parts[0], parts[-1]))
    k, v = (by_head(t, key_starts, lk) for t in parts[1:3])
    train = len(parts) > 3
    have, reach = key_starts.diff()[:, None], (key_starts.diff() - starts.diff())[:, None]
    limit = torch.minimum(((torch.arange(lq, device=dev) + reach) // frame + 1) * frame, have)
    hidden = (torch.arange(lk, device=dev) >= limit[..., None]).repeat(1, group, 1).repeat_interleave(kv, 0)
    results = [torch.empty_like(q)] + ([torch.empty_like(t) for t in (q, k, v)] if train else [])
    per = max(1, (1 << 30) // (group * lq * lk))      # heads at a time, so that the scores of a few fit
    for i in range(0, n * kv, per):
        part = slice(i, i + per)
        s = torch.matmul(q[part] * scale, k[part].transpose(-1, -2).contiguous()).masked_fill_(hidden[part], -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        p = p / p.sum(-1, keepdim=True).clamp_min(1e-37)
        results[0][part] = torch.matmul(p, v[part])
        if train:
            results[3][part] = torch.matmul(p.transpose(-1, -2).contiguous(), g[part])
            gp = torch.matmul(g[part], v[part].transpose(-1, -2).contiguous())
            gs = p * (gp - (p * gp).sum(-1, keepdim=True)) * scale
            results[1][part] = torch.matmul(gs, k[part])
            results[2][part] = torch.matmul(gs.transpose(-1, -2).contiguous(), q[part])
    return [back(r, s, m, like) for r, s, m, like in
            zip(results, (starts, starts, key_starts, key_starts), (lq, lq, lk, lk), (parts[0], parts[0], *parts[1:3]))]


def _plain_append(state):
    c, (k, v) = state["case"], state["inputs"]
    table, (lengths, seen), tokens = state["table"].long(), state["counts"].long(), state["tokens"]
    index = torch.arange(k.shape[0], device=k.device)
    if state["starts"] is None:
        stream, i, new = index, torch.zeros_like(index), torch.ones_like(lengths)
    else:
        starts = state["starts"].long()
        stream = torch.searchsorted(starts, index, right=True) - 1
        i, new = index - starts[stream], starts[1:] - starts[:-1]
    slot = lengths[stream] + i
    page, at = table[stream, slot // c["page"]], slot % c["page"]
    state["key"][page, :, at] = k
    state["value"][page, :, at] = v
    tokens[0][page, :, at] = 0
    tokens[1][page, :, at] = (seen[stream] + i).int()[:, None].expand(-1, c["kv_heads"])
    state["counts"].add_(new.int())
    return _memory_outputs(state)


def _slots(pages, table):
    """[pages, kv, page, ...] -> [n, kv, slots, ...]"""
    t = pages[table]
    return t.transpose(1, 2).flatten(2, 3)


def _plain_attend(state):
    c, q, table = state["case"], state["inputs"][0], state["table"].long()
    n, kv, group, lengths = c["n"], c["kv_heads"], c["heads"] // c["kv_heads"], state["counts"][0]
    k, v = (_slots(state[name], table).float() for name in ("key", "value"))
    s = torch.matmul(q.float().view(n, kv, group, -1) / math.sqrt(c["d"]), k.transpose(-1, -2).contiguous())
    hidden = torch.arange(k.shape[2], device=q.device) >= lengths[:, None]
    s = s.masked_fill_(hidden[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-37)
    out = torch.matmul(p, v).view(n, kv * group, -1).to(q.dtype)
    if not c["track"]:
        return out
    usage = state["tokens"][0].view(torch.float32)
    weight = p.sum(2).view(n, kv, -1, c["page"]).transpose(1, 2).flatten(0, 1)
    usage[table.flatten()] += weight
    return [out, usage]


def _plain_evict(state):
    c, table, keep = state["case"], state["table"].long(), state["case"]["keep"]
    lengths, seen = state["counts"]
    usage, positions = (_slots(t, table) for t in (state["tokens"][0].view(torch.float32), state["tokens"][1]))
    slot = torch.arange(usage.shape[2], device=usage.device)
    there = slot < lengths[:, None, None]
    rank = torch.where(positions >= (seen - c["recent"])[:, None, None], math.inf, usage)
    rank = torch.where(there, rank, -math.inf)
    kept = torch.empty_like(there.expand_as(rank))
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    kept.scatter_(-1, order, (slot < keep).expand_as(rank))
    kept = kept & there
    holes, fillers = there & ~kept & (slot < keep), kept & (slot >= keep)
    pairs = min(keep, max(usage.shape[2] - keep, 0))
    dst, src = (torch.sort((~t).byte(), dim=-1, stable=True).indices[..., :pairs] for t in (holes, fillers))
    src = torch.where(slot[:pairs] < holes.sum(-1, keepdim=True), src, dst)      # (no pair: a slot into itself)
    stream = torch.arange(c["n"], device=slot.device)[:, None, None]
    head = torch.arange(c["kv_heads"], device=slot.device)[:, None]
    to, of = ((table[stream, t // c["page"]], head, t % c["page"]) for t in (dst, src))
    for t in (state["key"], state["value"], state["tokens"][0], state["tokens"][1]):
        t[to] = t[of]
    lengths.clamp_(max=keep)
    return _memory_outputs(state)


# ---------------------------------------------------------------- in 64 bits, from the definitions
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"packed": _exact_packed, "append": _exact_append, "attend": _exact_attend, "evict": _exact_evict}[case["op"]](state)


def _exact_packed(state):
    c, (q, k, v) = state["case"], (t.detach().double() for t in state["inputs"])
    group, scale, train = c["heads"] // c["kv_heads"], 1.0 / math.sqrt(c["d"]), c["train"]
    grad = state["grad_out"].double() if train else None
    out, gq, gk, gv = (torch.zeros_like(t) for t in (q, q, k, v))
    q_end = k_end = 0
    for lq, lk in zip(*state["lengths"]):
        q_end, k_end = q_end + lq, k_end + lk
        if lq == 0:
            continue
        step = max(1, (1 << 28) // lk)
        for head in range(c["heads"]):
            at = slice(k_end - lk, k_end), head // group
            key, value = k[at].contiguous(), v[at].contiguous()
            for first in range(0, lq, step):
                count = min(step, lq - first)
                rows = slice(q_end - lq + first, q_end - lq + first + count), head
                # query number i is token lk - lq + i; it reads the frames up to its own
                token = torch.arange(first, first + count, device=q.device) + lk - lq
                frame_of_key = torch.arange(lk, device=q.device) // c["frame"]
                allowed = frame_of_key[None] <= (token // c["frame"])[:, None]
                query = q[rows].contiguous()
                s = (query @ key.t() * scale).masked_fill(~allowed, -math.inf)
                p = (s - torch.logsumexp(s, -1, keepdim=True)).exp()
                out[rows] = p @ value
                if train:
                    g = grad[rows].contiguous()
                    gv[at] += p.t() @ g
                    ds = p * (g @ value.t() - (g * out[rows]).sum(-1, keepdim=True)) * scale
                    gq[rows] = ds @ key
                    gk[at] += ds.t() @ query
    return [out, gq, gk, gv] if train else out


def _exact_append(state):
    c = state["case"]
    result = {name: t.double() if t.dtype.is_floating_point else t.clone() for name, t in _memory_outputs(state).items()}
    have, new, table = _lengths(c, c["longest"]), _new_lengths(c), state["table"].tolist()
    first = 0
    for n, (length, count) in enumerate(zip(have, new)):
        done = 0
        while done < count:      # a page at a time
            page, at = table[n][(length + done) // c["page"]], (length + done) % c["page"]
            some = min(c["page"] - at, count - done)
            rows = slice(first + done, first + done + some)
            for name, t in zip(("key", "value"), state["inputs"]):
                result[name][page, :, at:at + some] = t[rows].double().transpose(0, 1)
            result["usage"][page, :, at:at + some] = 0.0
            result["positions"][page, :, at:at + some] = length + 100 + done + torch.arange(some, device=state["key"].device).int()
            done += some
        first += count
        result["lengths"][n] = length + count
        result["seen"][n] = length + 100 + count
    return result


def _exact_attend(state):
    c, q = state["case"], state["inputs"][0].double()
    out = torch.zeros_like(q)
    usage = state["tokens"][0].view(torch.float32).double()
    group = c["heads"] // c["kv_heads"]
    for n, length in enumerate(_lengths(c, c["longest"])):
        if length == 0:
            continue
        slot = torch.arange(length, device=q.device)
        page, at = state["table"][n].long()[slot // c["page"]], slot % c["page"]
        for head in range(c["heads"]):
            s = (state["key"][page, head // group, at].double() * q[n, head]).sum(-1) / math.sqrt(c["d"])
            p = (s - torch.logsumexp(s, 0)).exp()
            out[n, head] = (p[:, None] * state["value"][page, head // group, at].double()).sum(0)
            usage[page, head // group, at] += p
    return [out, usage] if c["track"] else out


def _exact_evict(state):
    c = state["case"]
    result = {name: t.double() if t.dtype.is_floating_point else t.clone() for name, t in _memory_outputs(state).items()}
    dev, keep = state["key"].device, c["keep"]
    usage, positions = state["tokens"][0].view(torch.float32).cpu().numpy(), state["tokens"][1].cpu().numpy()
    table = state["table"].cpu().numpy()
    for n, length in enumerate(_lengths(c, c["longest"])):
        result["lengths"][n] = min(length, keep)
        if length <= keep:
            continue
        pages = table[n][:-(-length // c["page"])]
        for head in range(c["kv_heads"]):
            use = usage[pages, head].reshape(-1)[:length]
            newest = positions[pages, head].reshape(-1)[:length] >= length + 100 - c["recent"]
            stays = {int(i) for i in newest.nonzero()[0]}
            others = sorted((i for i in range(length) if i not in stays), key=lambda i: (-use[i], i))
            stays.update(others[:keep - len(stays)])
            holes = [i for i in range(keep) if i not in stays]
            fillers = sorted(i for i in stays if i >= keep)
            to, of = (torch.tensor(t, dtype=torch.long, device=dev) for t in (holes, fillers))
            place = state["table"][n].long()
            to, of = ((place[t // c["page"]], head, t % c["page"]) for t in (to, of))
            for name, t in _memory_outputs(state).items():
                if t.dim() > 1:
                    result[name][to] = t[of].to(result[name].dtype)
    return result
