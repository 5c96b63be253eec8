"""CrossAttention3d: the three operators as a network runs them, against the same block written out in float64; keys and values that
are kept between calls; what it refuses."""
import pytest
import torch
import torch.nn.functional as F

import d2conv3d_amd as d2c
from _util import rel_l2

pytestmark = pytest.mark.gpu


def turned(x, dims, pairs, base):
    """Rotary positions of [N, L, H, D] on a grid, in float64."""
    T, H, W = dims
    i = torch.arange(T * H * W)
    pos = torch.stack([i // (H * W), i // W % H, i % W], -1).double()
    angle = torch.cat([pos[:, a:a + 1] * base ** (-torch.arange(p).double() / p) for a, p in enumerate(pairs)], -1)[:, None]
    half = sum(pairs)
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    c, s = angle.cos(), angle.sin()
    return torch.cat([a * c - b * s, a * s + b * c, rest], -1)


def written_out(block, x, memory, mask):
    def tokens(t):
        return t.flatten(2).transpose(1, 2)

    def norm(m, t):
        return F.layer_norm(t, t.shape[-1:], m.weight.double(), m.bias.double(), m.eps)

    def linear(m, t):
        return F.linear(t, m.weight.double(), m.bias.double())
    N, d, h, kv = x.size(0), block.head_channels, block.heads, block.kv_heads
    q = linear(block.query, norm(block.norm, tokens(x))).view(N, -1, h, d)
    both = linear(block.key_value, norm(block.memory_norm, tokens(memory))).view(N, -1, 2, kv, d)
    q = turned(q, x.shape[2:], block.axis_pairs, block.base)
    k, v = turned(both[:, :, 0], memory.shape[2:], block.axis_pairs, block.base), both[:, :, 1]
    k, v = (t.repeat_interleave(h // kv, 2) for t in (k, v))
    s = torch.einsum("nqhd,nkhd->nhqk", q, k) / d ** 0.5
    if mask is not None:
        s = s.masked_fill(~mask.flatten(1)[:, None, None], float("-inf"))
    read = torch.einsum("nhqk,nkhd->nqhd", s.softmax(-1), v).flatten(2)
    return x + linear(block.out, read).transpose(1, 2).reshape(x.shape)


def make(dtype, kv_heads=2, memory_channels=48):
    torch.manual_seed(5)
    block = d2c.CrossAttention3d(64, heads=4, kv_heads=kv_heads, memory_channels=memory_channels)
    assert not bool(block.out.weight.any())
    for p in block.parameters():
        torch.nn.init.normal_(p, 0.0, 0.15)
    torch.nn.init.normal_(block.norm.weight, 1.0, 0.1)
    torch.nn.init.normal_(block.memory_norm.weight, 1.0, 0.1)
    block = block.to(dtype)
    return block, torch.randn(2, 64, 2, 5, 6).to(dtype), torch.randn(2, 48, 3, 6, 7).to(dtype)


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-5), (torch.bfloat16, 2e-2)])
def test_block_against_float64(dtype, tol, dev):
    block, x, memory = make(dtype)
    mask = torch.ones(2, 3, 6, 7, dtype=torch.bool)
    mask[0, 1], mask[1, :, :2] = False, False
    grad = torch.randn(x.shape).to(dtype)
    leaves = [x.double().requires_grad_(), memory.double().requires_grad_()]
    params = dict(block.named_parameters())
    want = written_out(block, *leaves, mask)
    wgrads = torch.autograd.grad(want, leaves + list(params.values()), grad.double())
    gpu = [x.to(dev).requires_grad_(), memory.to(dev).requires_grad_()]
    block = block.to(dev)
    out = block(*gpu, memory_mask=mask.to(dev))
    grads = torch.autograd.grad(out, gpu + list(block.parameters()), grad.to(dev))
    assert rel_l2(out, want) < tol
    for name, a, e in zip(["x", "memory", *params], grads, wgrads):
        if name == "key_value.bias":      # (the keys' half is 0 in exact arithmetic)
            half = a.numel() // 2
            a, e = a[half:], e[half:]
        assert rel_l2(a, e) < tol, (name, rel_l2(a, e))


def test_a_memory_kept_between_calls(dev):
    block, x, memory = make(torch.float32)
    block, x, memory = block.to(dev), x.to(dev), memory.to(dev)
    with torch.no_grad():
        kept = block.remember(memory)
        for frame in range(x.size(2)):
            one = x[:, :, frame:frame + 1].contiguous()
            assert torch.equal(block(one, kept), block(one, memory))
        frames = torch.tensor([[True, False, True], [False, True, True]], device=dev)
        cells = frames[:, :, None, None].expand(2, 3, 6, 7)
        assert torch.equal(block(x, kept, memory_mask=frames), block(x, kept, memory_mask=cells))
        lengths = torch.tensor([42, 84], device=dev)
        first = torch.arange(126, device=dev) < lengths[:, None]
        assert torch.equal(block(x, kept, memory_lengths=lengths), block(x, kept, memory_mask=first))
        assert torch.equal(block(x, kept, memory_lengths=torch.zeros(2, dtype=torch.int32, device=dev)),
                           x + block.out.bias.view(-1, 1, 1, 1))


def test_a_new_block_changes_nothing(dev):
    block = d2c.CrossAttention3d(32, heads=2).to(dev)
    x = torch.randn(1, 32, 2, 3, 4, device=dev)
    assert torch.equal(block(x, torch.randn(1, 32, 1, 5, 5, device=dev)), x)


def test_refusals(dev):
    for kw in (dict(heads=3), dict(heads=8, kv_heads=3)):
        with pytest.raises(ValueError, match="do not divide"):
            d2c.CrossAttention3d(64, **kw)
    with pytest.raises(ValueError, match="up to 128"):
        d2c.CrossAttention3d(512, heads=2)
    block = d2c.CrossAttention3d(32, heads=2).to(dev)
    with pytest.raises(RuntimeError, match="does not fit"):
        block(torch.zeros(1, 32, 1, 2, 2, device=dev), torch.zeros(1, 32, 3, 2, 2, device=dev),
              memory_mask=torch.ones(1, 5, dtype=torch.bool, device=dev))
