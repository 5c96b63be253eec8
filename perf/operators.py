"""What is timed of the operators that let a clip's feature map read the features of other frames: layer norm over the
channels of a position, rotary positions along time, height and width, and attention from the positions of one map to
those of another.  Inference (forward only) and a training step's share (forward and all gradients), float32 and
bfloat16.

A case is a dict of plain values:

  op        "layer_norm" | "rotary" | "attention"
  dtype     "f32" | "bf16": element type of the inputs, the outputs and their gradients
  train     forward and all gradients; otherwise forward only
  n         samples (clips)

  layer_norm: rows (positions of a sample), c (channels), params ("f32" | "bf16": type of weight and bias)
  rotary:     t, h, w (the map), heads, d, source ("grid": positions are the map's indices; "tensor": real positions of
              each token), interleaved
  attention:  lq, lk (positions that read, positions that are read), heads, kv_heads, d,
              mask ("none"; "lengths": each sample has its own number of keys; "frames": whole frames of the memory are
              not to be read; "mixed": both), fill (about which share of the keys is read),
              packed (keys and values lie in one buffer, as a common projection leaves them)
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-5
BASE = 10000.0


# ---------------------------------------------------------------- cases
def _norm(n, rows, c, dtype, train, params="f32"):
    return dict(op="layer_norm", n=n, rows=rows, c=c, dtype=dtype, train=train, params=params)


def _rotary(n, t, h, w, heads, d, dtype, train, source="grid", interleaved=False):
    return dict(op="rotary", n=n, t=t, h=h, w=w, heads=heads, d=d, dtype=dtype, train=train, source=source,
                interleaved=interleaved)


def _attention(n, lq, lk, heads, kv_heads, d, dtype, train, mask="none", fill=1.0, packed=False):
    return dict(op="attention", n=n, lq=lq, lk=lk, heads=heads, kv_heads=kv_heads, d=d, dtype=dtype, train=train,
                mask=mask, fill=fill, packed=packed)


def listed():
    cases = {
        # one small frame in inference, an odd number of channels: launches and host work count
        "norm small frame f32 infer": _norm(1, 350, 257, "f32", False),
        # the positions of two clips at stride 16, a training step in mixed precision
        "norm decoder bf16 train": _norm(2, 12960, 512, "bf16", True),
        # a long clip at stride 8
        "norm long clip bf16 train": _norm(1, 207360, 256, "bf16", True, "bf16"),
        # queries of one small frame
        "rotary small frame bf16 infer": _rotary(1, 1, 14, 25, 8, 64, "bf16", False),
        # the keys of two remembered clips with their real positions, a head size that is no power of two
        "rotary positions f32 train": _rotary(2, 8, 30, 54, 4, 80, "f32", True, "tensor", True),
        # a long clip at stride 8
        "rotary long clip bf16 train": _rotary(1, 32, 60, 108, 8, 64, "bf16", True),
        # one token that sums up a clip, keys shared by four heads each: serving, one token at a time
        "attention one token bf16 infer": _attention(1, 1, 12960, 16, 4, 64, "bf16", False, packed=True),
        # object queries read the memories of three clips, each of its own length
        "attention object queries f32 infer": _attention(3, 100, 3240, 8, 8, 32, "f32", False, "lengths", 0.7),
        # odd sizes in float32, a training step
        "attention odd f32 train": _attention(1, 1417, 3001, 6, 3, 40, "f32", True),
        # a frame reads its clip, some frames of which are not to be read
        "attention frame to clip bf16 train": _attention(2, 1620, 12960, 8, 8, 64, "bf16", True, "frames", 0.75),
        # a frame reads a long memory, keys and values shared by four heads each
        "attention long memory bf16 infer": _attention(1, 1620, 64800, 8, 2, 128, "bf16", False, packed=True),
        # every position of a clip reads every position of two clips
        "attention clip to clips bf16 train": _attention(1, 12960, 25920, 8, 8, 64, "bf16", True),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    largest = {}
    for c in listed():
        largest[c["op"]] = max(largest.get(c["op"], 0.0), _weight(c))
    while True:
        op = rng.choice(["layer_norm", "rotary", "attention", "attention"])
        dtype = rng.choice(["f32", "bf16"])
        train = rng.random() < 0.6
        n = rng.choice([1, 1, 2, 3, 4])
        if op == "layer_norm":
            c = rng.choice([_log_int(rng, 16, 2048), rng.choice([64, 128, 256, 512, 1024, 2048])])
            case = _norm(n, _log_int(rng, 1, 207360), c, dtype, train, rng.choice(["f32", dtype]))
        elif op == "rotary":
            h = _log_int(rng, 7, 64)
            case = _rotary(n, _log_int(rng, 1, 32), h, max(7, round(h * rng.uniform(0.9, 1.9))),
                           rng.choice([1, 2, 4, 6, 8, 16]), rng.choice([24, 32, 40, 64, 64, 80, 96, 128]), dtype, train,
                           rng.choice(["grid", "tensor"]), rng.random() < 0.5)
        else:
            kv_heads = rng.choice([1, 2, 3, 4, 8])
            mask = rng.choice(["none", "none", "lengths", "frames", "mixed"])
            case = _attention(n, _log_int(rng, 1, 12960), _log_int(rng, 1, 64800), kv_heads * rng.choice([1, 1, 2, 4]),
                              kv_heads, rng.choice([24, 32, 40, 64, 64, 80, 96, 128, 128]), dtype, train, mask,
                              1.0 if mask == "none" else round(rng.uniform(0.2, 0.9), 2), rng.random() < 0.4)
        if _weight(case) <= largest[op]:
            return case


def _pairs(d):
    """Pairs of a head's channels that turn with time, height and width: the whole head, time a little less."""
    side = (d // 2 * 3 + 4) // 8
    return d // 2 - 2 * side, side, side


def _elements(case):
    """Elements read and written in the case's element type, and elements of 4 bytes."""
    c, n = case, case["n"]
    if c["op"] == "layer_norm":
        x, params = n * c["rows"] * c["c"], 2 * c["c"]
        wide = c["params"] == "f32"
        params *= 2 if c["train"] else 1
        return (4 if c["train"] else 2) * x + (0 if wide else params), params if wide else 0
    if c["op"] == "rotary":
        tokens = n * c["t"] * c["h"] * c["w"]
        x = tokens * c["heads"] * c["d"]
        return (4 if c["train"] else 2) * x, 3 * tokens if c["source"] == "tensor" else 0
    q = n * c["lq"] * c["heads"] * c["d"]
    kv = 2 * n * c["lk"] * c["kv_heads"] * c["d"]
    if c["train"]:
        return 4 * q + kv * c["fill"] + kv, 0
    return 2 * q + kv * c["fill"], 0


def work(case):
    c = case
    moved, words = _elements(c)
    size = 2 if c["dtype"] == "bf16" else 4
    if c["op"] == "layer_norm":
        flops = 8.0 * c["n"] * c["rows"] * c["c"] * (3 if c["train"] else 1)
    elif c["op"] == "rotary":
        flops = 3.0 * c["n"] * c["t"] * c["h"] * c["w"] * c["heads"] * c["d"] * (2 if c["train"] else 1)
    else:
        flops = 4.0 * c["n"] * c["lq"] * c["lk"] * c["fill"] * c["heads"] * c["d"] * (3.5 if c["train"] else 1)
    return {"bytes": float(moved * size + words * 4), "flops": flops}


def _weight(c):
    """How much a case costs, roughly (a float32 product counts like six)."""
    w = work(c)
    return w["bytes"] + (w["flops"] * (6 if c["dtype"] == "f32" else 1) / 100 if c["op"] == "attention" else 0)


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    c, dev, dtype = case, torch.device("cuda"), DTYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    n, train = c["n"], c["train"]

    def normal(*shape, std=1.0, mean=0.0, type=dtype):
        return (torch.randn(*shape, generator=gen, device=dev) * std + mean).to(type)

    state = {"case": c}
    if c["op"] == "layer_norm":
        kind = DTYPES[c["params"]]
        # features of a residual stream: each position with its own mean and spread
        x = normal(n, c["rows"], c["c"], type=torch.float32)
        x = x * normal(n, c["rows"], 1, std=0.3, mean=1.5, type=torch.float32)
        x = (x + normal(n, c["rows"], 1, std=0.5, type=torch.float32)).to(dtype)
        inputs = [x, normal(c["c"], std=0.2, mean=1.0, type=kind), normal(c["c"], std=0.2, type=kind)]
        out_shape = x.shape
    elif c["op"] == "rotary":
        tokens = c["t"] * c["h"] * c["w"]
        inputs = [normal(n, tokens, c["heads"], c["d"])]
        out_shape = inputs[0].shape
        if c["source"] == "tensor":
            # frames of a longer video, some left out, and cells' centres on the finest map
            start = torch.randint(0, 200, (n, 1), generator=gen, device=dev)
            step = torch.randint(1, 4, (n, c["t"]), generator=gen, device=dev).cumsum(1) + start
            rows = torch.arange(c["h"], device=dev) * 2 + 0.5
            cols = torch.arange(c["w"], device=dev) * 2 + 0.5
            grid = torch.empty(n, c["t"], c["h"], c["w"], 3, device=dev)
            grid[..., 0] = step[:, :, None, None]
            grid[..., 1] = rows[:, None]
            grid[..., 2] = cols
            state["positions"] = grid.view(n, tokens, 3)
        else:
            state["positions"] = (c["t"], c["h"], c["w"])
    else:
        lq, lk, kv = c["lq"], c["lk"], c["kv_heads"]
        q = normal(n, lq, c["heads"], c["d"])
        if c["packed"]:
            both = normal(n, lk, 2, kv, c["d"])
            inputs = [q, both[:, :, 0], both[:, :, 1]]
        else:
            inputs = [q, normal(n, lk, kv, c["d"]), normal(n, lk, kv, c["d"])]
        out_shape = q.shape
        share = math.sqrt(c["fill"]) if c["mask"] == "mixed" else c["fill"]
        state["lengths"] = state["key_mask"] = None
        if c["mask"] in ("lengths", "mixed"):
            spread = min(share, 1.0 - share) * (torch.rand(n, generator=gen, device=dev) * 2 - 1)
            state["lengths"] = ((share + spread) * lk).round().int().clamp_(0, lk)
        if c["mask"] in ("frames", "mixed"):
            frames = min(lk, 16)
            keep = torch.rand(n, frames, generator=gen, device=dev) < share
            frame = torch.arange(lk, device=dev) * frames // lk
            state["key_mask"] = keep[:, frame].contiguous()
    state["inputs"] = [v.requires_grad_(train) for v in inputs]
    if train:
        state["grad_out"] = normal(*out_shape)
    return state


# ---------------------------------------------------------------- the operators
def run(state):
    c = state["case"]
    if not own:
        with torch.no_grad():
            return _PLAIN[c["op"]](state)
    if not c["train"]:
        with torch.no_grad():
            return _call(state)
    out = _call(state)
    return [out.detach(), *torch.autograd.grad(out, state["inputs"], state["grad_out"])]


def _call(state):
    import d2conv3d_amd as d2c
    c, inputs = state["case"], state["inputs"]
    if c["op"] == "layer_norm":
        return d2c.layer_norm(*inputs, eps=EPS)
    if c["op"] == "rotary":
        return d2c.rotary3d(inputs[0], state["positions"], axis_pairs=_pairs(c["d"]), base=BASE,
                            interleaved=c["interleaved"])
    return d2c.cross_attention(*inputs, key_lengths=state["lengths"], key_mask=state["key_mask"])


def _plain_layer_norm(state):
    x, weight, bias = state["inputs"]
    v, w, b = x.float(), weight.float(), bias.float()
    mean = v.mean(-1, keepdim=True)
    centred = v - mean
    rstd = 1.0 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    hat = centred * rstd
    y = (hat * w + b).to(x.dtype)
    if not state["case"]["train"]:
        return y
    g = state["grad_out"].float()
    gw = g * w
    gx = rstd * (gw - gw.mean(-1, keepdim=True) - hat * (gw * hat).mean(-1, keepdim=True))
    return [y, gx.to(x.dtype), (g * hat).sum((0, 1)).to(weight.dtype), g.sum((0, 1)).to(bias.dtype)]


def _positions(state, dtype):
    p, dev = state["positions"], state["inputs"][0].device
    if isinstance(p, torch.Tensor):
        return p.to(dtype)
    t, h, w = p
    i = torch.arange(t * h * w, device=dev)
    return torch.stack([i // (h * w), i // w % h, i % w], -1).to(dtype)[None]


def _turn(x, cos, sin, interleaved):
    """Channel pairs of x [..., 2 * pairs], turned."""
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)


def _plain_rotary(state):
    c, x = state["case"], state["inputs"][0]
    pos = _positions(state, torch.float32)
    angles = []
    for axis, pairs in enumerate(_pairs(c["d"])):
        rate = torch.exp(torch.arange(pairs, device=x.device).float() * (-math.log(BASE) / pairs))
        angles.append(pos[..., axis:axis + 1] * rate)
    angle = torch.cat(angles, -1)[:, :, None]
    cos, sin = torch.cos(angle), torch.sin(angle)
    y = _turn(x.float(), cos, sin, c["interleaved"]).to(x.dtype)
    if not c["train"]:
        return y
    return [y, _turn(state["grad_out"].float(), cos, -sin, c["interleaved"]).to(x.dtype)]


def _allowed(state):
    """[N, Lk] truth values of the keys that are read, or None."""
    lengths, mask, k = state["lengths"], state["key_mask"], state["inputs"][1]
    if lengths is not None:
        below = torch.arange(k.shape[1], device=k.device) < lengths[:, None]
        mask = below if mask is None else mask & below
    return mask


def _plain_attention(state):
    c, (q, k, v) = state["case"], state["inputs"]
    n, lq, heads, d = q.shape
    lk, kv = k.shape[1], k.shape[2]
    group, scale = heads // kv, 1.0 / math.sqrt(d)

    def by_head(x):     # [N, L, kv * s, D] -> [N, kv, s * L, D]
        s = x.shape[2] // kv
        return x.float().view(n, x.shape[1], kv, s, d).permute(0, 2, 3, 1, 4).reshape(n, kv, s * x.shape[1], d)

    def back(x, like):  # ... and back
        s = like.shape[2] // kv
        return (x.view(n, kv, s, like.shape[1], d).permute(0, 3, 1, 2, 4).reshape(like.shape)).to(like.dtype)

    qh, kh, vh = by_head(q), by_head(k), by_head(v)
    allowed = _allowed(state)
    train = c["train"]
    gh = by_head(state["grad_out"]) if train else None
    out = torch.empty_like(qh)
    gq, gk, gv = (torch.empty_like(t) for t in (qh, kh, vh)) if train else (None,) * 3
    # heads at a time, so that the scores of a few fit
    per = max(1, (1 << 30) // (n * group * lq * lk))
    for i in range(0, kv, per):
        part = slice(i, i + per)
        key, value = kh[:, part], vh[:, part]
        s = torch.matmul(qh[:, part] * scale, key.transpose(-1, -2).contiguous())
        if allowed is not None:
            s = s.masked_fill(~allowed[:, None, None], -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        p = p / p.sum(-1, keepdim=True).clamp_min(1e-37)
        out[:, part] = torch.matmul(p, value)
        if train:
            g = gh[:, part]
            gv[:, part] = torch.matmul(p.transpose(-1, -2).contiguous(), g)
            gp = torch.matmul(g, value.transpose(-1, -2).contiguous())
            gs = p * (gp - (p * gp).sum(-1, keepdim=True)) * scale
            gq[:, part] = torch.matmul(gs, key)
            gk[:, part] = torch.matmul(gs.transpose(-1, -2).contiguous(), qh[:, part])
    if not train:
        return back(out, q)
    return [back(out, q), back(gq, q), back(gk, k), back(gv, v)]


_PLAIN = {"layer_norm": _plain_layer_norm, "rotary": _plain_rotary, "attention": _plain_attention}


# ---------------------------------------------------------------- in 64 bits, from the definitions
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"layer_norm": _exact_layer_norm, "rotary": _exact_rotary, "attention": _exact_attention}[case["op"]](state)


def _exact_layer_norm(state):
    x, w, b = (t.detach().double() for t in state["inputs"])
    var, mean = torch.var_mean(x, -1, unbiased=False, keepdim=True)
    std = (var + EPS).sqrt()
    y = (x - mean) / std * w + b
    if not state["case"]["train"]:
        return y
    g = state["grad_out"].double()
    # y = f(x) per row: the Jacobian of (x - mean) / std applied to g * w
    size = x.shape[-1]
    u = g * w
    centred = x - mean
    gx = (u - u.sum(-1, keepdim=True) / size) / std - centred * (u * centred).sum(-1, keepdim=True) / (size * std ** 3)
    return [y, gx, (g * (centred / std)).flatten(0, 1).sum(0), g.flatten(0, 1).sum(0)]


def _exact_rotary(state):
    c, x = state["case"], state["inputs"][0].detach().double()
    pos = _positions(state, torch.float64)
    d, pairs = c["d"], _pairs(c["d"])

    def turned(x, sign):
        y = x.clone()
        j = 0
        for axis in range(3):
            for i in range(pairs[axis]):
                a, b = (2 * j, 2 * j + 1) if c["interleaved"] else (j, j + sum(pairs))
                angle = sign * pos[..., axis] * BASE ** (-i / pairs[axis])
                cos, sin = torch.cos(angle)[..., None], torch.sin(angle)[..., None]
                y[..., a] = x[..., a] * cos - x[..., b] * sin
                y[..., b] = x[..., a] * sin + x[..., b] * cos
                j += 1
        return y

    assert 2 * sum(pairs) <= d
    return [turned(x, 1.0), turned(state["grad_out"].double(), -1.0)] if c["train"] else turned(x, 1.0)


def _exact_attention(state):
    c, (q, k, v) = state["case"], (t.detach().double() for t in state["inputs"])
    n, lq, heads, d = q.shape
    group = heads // k.shape[2]
    allowed = _allowed(state)
    g = state["grad_out"].double() if c["train"] else None
    out = torch.zeros_like(q)
    grads = [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in (q, k, v)]
    rows = max(1, (1 << 28) // k.shape[1])
    for b in range(n):
        keys = slice(None) if allowed is None else allowed[b].nonzero()[:, 0]
        for head in range(heads):
            key, value = k[b, keys, head // group].contiguous(), v[b, keys, head // group].contiguous()
            if key.shape[0] == 0:
                continue
            gk, gv = torch.zeros_like(key), torch.zeros_like(value)
            for i in range(0, lq, rows):
                part = slice(i, i + rows)
                query = q[b, part, head].contiguous()
                s = query @ key.t() / math.sqrt(d)
                p = (s - torch.logsumexp(s, -1, keepdim=True)).exp()
                out[b, part, head] = p @ value
                if c["train"]:
                    go = g[b, part, head].contiguous()
                    gv += p.t() @ go
                    gs = p * (go @ value.t() - (go * out[b, part, head]).sum(-1, keepdim=True)) / math.sqrt(d)
                    grads[0][b, part, head] = gs @ key
                    gk += gs.t() @ query
            if c["train"]:
                grads[1][b, keys, head // group] += gk
                grads[2][b, keys, head // group] += gv
    return [out, *grads] if c["train"] else out
