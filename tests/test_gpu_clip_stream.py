"""The operators as a network uses them: trained on packed clips, serving the same tokens one at a time from a memory in pages."""
import math

import pytest
import torch

import d2conv3d_amd as d2c

pytestmark = pytest.mark.gpu

H, KV, D, C = 4, 2, 64, 256
FRAME = (3, 4)                    # cells of a frame
CELLS = FRAME[0] * FRAME[1]


class Block(torch.nn.Module):
    """x + out(attention(rotary(q(norm(x))), rotary(k(norm(x))), v(norm(x)))), causal, over packed clips or one token at a time"""

    def __init__(self):
        super().__init__()
        self.norm = d2c.LayerNorm(C)
        self.qkv = torch.nn.Linear(C, (H + 2 * KV) * D)
        self.out = torch.nn.Linear(H * D, C)

    def project(self, x, positions):
        qkv = self.qkv(self.norm(x)).view(1, x.shape[0], H + 2 * KV, D)
        turned = d2c.rotary3d(qkv[:, :, :H + KV], positions[None])[0]
        return turned[:, :H], turned[:, H:], qkv[0, :, H + KV:]

    def forward(self, x, starts, positions):
        read = d2c.packed_attention(*self.project(x, positions), starts)
        return x + self.out(read.flatten(1))

    def step(self, x, memory, positions, track=False):
        q, k, v = self.project(x, positions)
        memory.append(k, v)
        return x + self.out(memory.attend(q, track=track).flatten(1))


def places(lengths, dev):
    """(frame, row, column) of every token of the clips"""
    t = torch.cat([torch.arange(n) for n in lengths]).to(dev)
    return torch.stack([t // CELLS, t % CELLS // FRAME[1], t % FRAME[1]], -1).float()


def plain(block, x, lengths, positions):
    """The block in elementary operations and 64 bits, clip by clip"""
    x = x.double()
    mean, var = x.mean(-1, keepdim=True), x.var(-1, unbiased=False, keepdim=True)
    y = (x - mean) / (var + block.norm.eps).sqrt() * block.norm.weight.double() + block.norm.bias.double()
    qkv = (y @ block.qkv.weight.double().t() + block.qkv.bias.double()).view(-1, H + 2 * KV, D)
    angle = []
    for axis, pairs in enumerate((8, 12, 12)):
        rate = 10000.0 ** (-torch.arange(pairs, device=x.device).double() / pairs)
        angle.append(positions[:, axis:axis + 1].double() * rate)
    cos, sin = (f(torch.cat(angle, -1))[:, None] for f in (torch.cos, torch.sin))
    a, b = qkv[:, :H + KV, :D // 2], qkv[:, :H + KV, D // 2:]
    turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    outs, first = [], 0
    for n in lengths:
        at = slice(first, first + n)
        first += n
        q, k, v = turned[at, :H].transpose(0, 1), turned[at, H:].transpose(0, 1).repeat_interleave(H // KV, 0), qkv[at, H + KV:].transpose(0, 1).repeat_interleave(H // KV, 0)
        s = (q @ k.transpose(1, 2).contiguous() / math.sqrt(D)).masked_fill(torch.ones(n, n, device=x.device).triu(1).bool(), -math.inf)
        outs.append((torch.softmax(s, -1) @ v).transpose(0, 1).reshape(n, H * D))
    return x + torch.cat(outs) @ block.out.weight.double().t() + block.out.bias.double()


def test_default_pairs():
    from d2conv3d_amd.attention import default_axis_pairs
    assert default_axis_pairs(D) == (8, 12, 12)


def test_trained_on_packed_clips(dev):
    """Output and every gradient of a training step against 64 bits, float32: a few hundred float32 operations in a row of each, 1e-5 of the largest"""
    torch.manual_seed(1)
    block, lengths = Block().to(dev), [40, 0, 1, 130]
    starts = torch.tensor([0] + lengths, device=dev).cumsum(0)
    x = torch.randn(sum(lengths), C, device=dev, requires_grad=True)
    g = torch.randn(sum(lengths), C, device=dev)
    positions = places(lengths, dev)
    leaves = [x, *block.parameters()]
    out = block(x, starts, positions)
    grads = torch.autograd.grad(out, leaves, g)
    want = plain(block, x, lengths, positions)
    exact = torch.autograd.grad(want, leaves, g.double())
    for a, b in zip((out, *grads), (want, *exact)):
        assert (a.double() - b.double()).abs().max() <= 1e-5 * b.double().abs().max()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_served_token_by_token(dtype, dev):
    """A clip's first tokens at once, the others one at a time: what the packed call makes of the whole clips.  Tolerances: float32 as above; bfloat16 rounds six
    times between a token and its output (norm, projection, turn, attention, projection, sum), 2^-8 each of values of about 1, and the weights: 8 * 2^-8 of the largest"""
    torch.manual_seed(2)
    block, lengths, given = Block().to(dev, dtype), [30, 90, 7], [12, 60, 0]
    tolerance = 1e-5 if dtype == torch.float32 else 8 * 2.0 ** -8
    starts = torch.tensor([0] + lengths, device=dev).cumsum(0).int()
    x = torch.randn(sum(lengths), C, device=dev, dtype=dtype)
    positions = places(lengths, dev)
    with torch.no_grad():
        whole = block(x, starts, positions)
        memory = d2c.PagedMemory.empty(3, 100, KV, D, page=16, dtype=dtype, device=dev)
        # the clips' beginnings, packed
        index = torch.cat([torch.arange(n) + s for n, s in zip(given, starts.tolist())]).to(dev)
        some = torch.tensor([0] + given, device=dev).cumsum(0).int()
        q, k, v = block.project(x[index], positions[index])
        memory.append(k, v, some)
        begun = x[index] + block.out(d2c.packed_attention(q, k, v, some).flatten(1))
        limit = tolerance * whole.double().abs().max()
        assert (begun.double() - whole[index].double()).abs().max() <= limit
        # ... and the rest, each stream as long as its clip lasts
        for t in range(max(n - m for n, m in zip(lengths, given))):
            at = torch.tensor([min(m + t, n - 1) + s for n, m, s in zip(lengths, given, starts.tolist())], device=dev)
            y = block.step(x[at], memory, positions[at])
            live = torch.tensor([m + t < n for n, m in zip(lengths, given)], device=dev)
            assert ((y.double() - whole[at].double()).abs().amax(-1)[live] <= limit).all(), t
    assert memory.seen.tolist() == [12 + t + 1, 60 + t + 1, t + 1]


def test_a_piece_behind_what_is_there(dev):
    """A clip that goes on: the new piece's queries against keys of the whole."""
    torch.manual_seed(3)
    block, lengths, given = Block().to(dev), [50, 33], [20, 33]
    starts = torch.tensor([0] + lengths, device=dev).cumsum(0).int()
    x, positions = torch.randn(sum(lengths), C, device=dev), places(lengths, dev)
    with torch.no_grad():
        whole = block(x, starts, positions)
        q, k, v = block.project(x, positions)
        index = torch.cat([torch.arange(m, n) + s for n, m, s in zip(lengths, given, starts.tolist())]).to(dev)
        some = torch.tensor([0, 30, 30], device=dev).int()
        y = x[index] + block.out(d2c.packed_attention(q[index], k, v, some, starts).flatten(1))
    assert (y.double() - whole[index].double()).abs().max() <= 1e-5 * whole.double().abs().max()


def test_a_stream_that_forgets(dev):
    """Weights are added up while a stream is read, its memory is kept at a size: what stays are the newest tokens and those that were read most, and what is read
    then is attention over what stayed."""
    torch.manual_seed(4)
    block, n, keep, recent = Block().to(dev), 2, 24, 6
    memory = d2c.PagedMemory.empty(n, 40, KV, D, page=8, dtype=torch.float32, device=dev)
    kept = [[[] for _ in range(KV)] for _ in range(n)]      # (position, key, value, usage) in 64 bits
    with torch.no_grad():
        for t in range(60):
            x, positions = torch.randn(n, C, device=dev), torch.full((n, 3), float(t), device=dev)
            q, k, v = block.project(x, positions)
            memory.append(k, v)
            out = memory.attend(q, track=True)
            for i in range(n):
                for h in range(KV):
                    mine = kept[i][h]
                    mine.append([t, k[i, h].double(), v[i, h].double(), 0.0])
                    keys, values = (torch.stack([m[j] for m in mine]) for j in (1, 2))
                    p = torch.softmax(q[i, h * 2:h * 2 + 2].double() @ keys.t() / math.sqrt(D), -1)
                    assert (out[i, h * 2:h * 2 + 2].double() - p @ values).abs().max() < 1e-5
                    for m, u in zip(mine, p.sum(0).tolist()):
                        m[3] += u
            if memory.lengths[0].item() > 32:
                memory.evict(keep, recent)
                for i in range(n):
                    for h in range(KV):
                        mine = kept[i][h]
                        old = sorted((m for m in mine if m[0] < t + 1 - recent), key=lambda m: -m[3])
                        # (no two usages as near as float32 sums are off: the border is clear)
                        assert old[keep - recent - 1][3] - old[keep - recent][3] > 1e-5
                        kept[i][h] = old[:keep - recent] + [m for m in mine if m[0] >= t + 1 - recent]
                        slots = memory.lengths[i].item()
                        page = memory.table[i].long()[torch.arange(slots, device=dev) // 8]
                        there = memory.positions[page, h, torch.arange(slots, device=dev) % 8]
                        assert sorted(there.tolist()) == sorted(m[0] for m in kept[i][h])
    assert memory.seen.tolist() == [60, 60]


def test_in_inference_mode(dev):
    with torch.inference_mode():
        memory = d2c.PagedMemory.empty(1, 20, KV, D, device=dev)
        t = torch.randn(1, KV, D, device=dev).bfloat16()
        memory.append(t, t)
        assert torch.equal(memory.attend(t, track=True), t)
        memory.evict(1)
    assert memory.lengths.tolist() == [1]
