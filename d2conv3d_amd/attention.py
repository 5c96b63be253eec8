"""A map's positions read another map's: layer norm over the channels of a position, rotary positions along time, height
and width, attention to positions of another number, and the block of a network that they make up.  (No counterpart in
the reference, whose decoder joins the features of different frames by convolutions alone.)

    layer_norm        torch.nn.functional.layer_norm over the last dimension
    rotary3d          rotary position embedding with three axes
    cross_attention   softmax(scale q k^T) v over the keys that are there, query heads sharing key heads
    CrossAttention3d  the block: a clip's feature map reads the feature map of remembered frames

float32 and bfloat16 run as they are (sums and statistics in float32); float16 is computed in float32 and returned as
float16.
"""
import ctypes
import math

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable
from torch.utils._pytree import register_pytree_node

from . import _lib
from ._ops import _DT, _ptr, _stream, _try_native, _workspace

_TYPES = (torch.float32, torch.bfloat16)


def _check(cond, msg):
    if not cond:
        raise RuntimeError(msg)


def _check_tensors(what, **tensors):
    """Tensors on one GPU, of types that the kernels (or their float16 detour) take."""
    first = None
    for name, t in tensors.items():
        if t is None:
            continue
        _check(isinstance(t, torch.Tensor), f"{what}: {name} must be a Tensor")
        if not t.is_cuda:
            raise RuntimeError(f"{what}: {name} must be on the GPU (this build has no CPU path)")
        first = t if first is None else first
        _check(t.device == first.device, f"{what}: {name} is on {t.device}, the first tensor on {first.device}")


def _long3(*v):
    return (ctypes.c_int64 * 3)(*v)


# ---------------------------------------------------------------- layer norm
def _rows(x):
    """[rows, channels], in place where the rows lie at one distance, and that distance."""
    x = x.reshape(-1, x.size(-1))
    if x.stride(1) != 1 and x.size(1) > 1:
        x = x.contiguous()
    return x, x.stride(0)


class _LayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, weight, bias, eps):
        lib, dev, C = _lib.load(), input.device, input.size(-1)
        x, stride = _rows(input)
        params = weight if weight is not None else bias
        desc = _lib.LayerNormDesc(x.size(0), stride, C, _DT[x.dtype], _DT[(x if params is None else params).dtype], eps)
        out = torch.empty(input.shape, dtype=x.dtype, device=dev)
        w = None if weight is None else weight.contiguous()
        b = None if bias is None else bias.contiguous()
        stats = torch.empty((x.size(0), 2), dtype=torch.float32, device=dev) if any(ctx.needs_input_grad) else None
        with torch.cuda.device(dev):
            rc = lib.d2c_layer_norm_forward(ctypes.byref(desc), _ptr(x), _ptr(w), _ptr(b), _ptr(out), _ptr(stats), _stream(dev))
        _lib.check(rc, "layer_norm forward")
        # (the input itself where its rows are read in place: a view made here would hide the input's version from autograd)
        ctx.save_for_backward(input if x.data_ptr() == input.data_ptr() else x, w, b, stats)
        ctx.desc, ctx.shape = desc, input.shape
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        lib = _lib.load()
        x, w, b, stats = ctx.saved_tensors
        desc, dev, need = ctx.desc, x.device, ctx.needs_input_grad
        x, desc.x_stride = _rows(x)      # (strides of what came back: hooks of the caller may have put it elsewhere in the meantime)
        g = grad_out.to(x.dtype).contiguous()
        gx = torch.empty(ctx.shape, dtype=x.dtype, device=dev) if need[0] else None
        gw = torch.empty_like(w) if w is not None and need[1] else None
        gb = torch.empty_like(b) if b is not None and need[2] else None
        with torch.cuda.device(dev):
            nb = lib.d2c_layer_norm_backward_workspace_bytes(ctypes.byref(desc)) if gw is not None or gb is not None else 0
            ws = _workspace(nb, dev)
            rc = lib.d2c_layer_norm_backward(ctypes.byref(desc), _ptr(g), _ptr(x), _ptr(stats), _ptr(w), _ptr(gx), _ptr(gw),
                                             _ptr(gb), _ptr(ws), nb, _stream(dev))
        _lib.check(rc, "layer_norm backward")
        return gx, gw, gb, None


def layer_norm(input, weight=None, bias=None, eps=1e-5):
    """`torch.nn.functional.layer_norm(input, input.shape[-1:], weight, bias, eps)`: up to 16384 channels; rows of any
    distance from each other are read in place.  `weight` and `bias` [channels] may be None and may be float32 beside a
    bfloat16 input.  Gradients of all three; statistics and the sums of the gradients are held in float32."""
    out = _try_native("layer_norm", input, weight, bias, eps)
    if out is not None:
        return out
    _check_tensors("layer_norm", input=input, weight=weight, bias=bias)
    _check(input.dim() >= 1 and input.size(-1) > 0, "layer_norm: input needs a last dimension with channels")
    for name, t in (("weight", weight), ("bias", bias)):
        _check(t is None or tuple(t.shape) == (input.size(-1),),
               f"layer_norm: {name} must have the shape ({input.size(-1)},), got {None if t is None else tuple(t.shape)}")
    if input.dtype == torch.float16:
        return layer_norm(input.float(), None if weight is None else weight.float(), None if bias is None else bias.float(),
                          eps).half()
    _check(input.dtype in _TYPES, f"layer_norm: unsupported dtype {input.dtype}")
    if any(t is not None and t.dtype != input.dtype for t in (weight, bias)):
        weight, bias = (None if t is None else t.float() for t in (weight, bias))
    return _LayerNormFunction.apply(input, weight, bias, float(eps))


# ---------------------------------------------------------------- rotary positions
def _rotary_call(x, positions, grid, pairs, base, interleaved, direction):
    if x.stride(3) != 1 and x.size(3) > 1:
        x = x.contiguous()
    N, L, H, D = x.shape
    desc = _lib.Rotary3dDesc(N, L, H, D, (ctypes.c_int32 * 3)(*pairs), (ctypes.c_int32 * 3)(*grid), int(interleaved), direction,
                             _DT[x.dtype], base, _long3(*x.stride()[:3]),
                             0 if positions is None or positions.dim() == 2 else positions.stride(0))
    out = torch.empty((N, L, H, D), dtype=x.dtype, device=x.device)
    with torch.cuda.device(x.device):
        rc = _lib.load().d2c_rotary3d(ctypes.byref(desc), _ptr(x), _ptr(positions), _ptr(out), _stream(x.device))
    _lib.check(rc, "rotary3d")
    return out


class _Rotary3dFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, positions, *geometry):
        ctx.save_for_backward(positions)
        ctx.geometry = geometry
        return _rotary_call(input, positions, *geometry, 1)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        return (_rotary_call(grad_out, ctx.saved_tensors[0], *ctx.geometry, -1),) + (None,) * 5


def default_axis_pairs(head_channels):
    """Channel pairs of a head that turn with time, height and width: all of them, height and width 3/8 each."""
    side = (head_channels // 2 * 3 + 4) // 8
    return head_channels // 2 - 2 * side, side, side


def rotary3d(input, positions, axis_pairs=None, base=10000.0, interleaved=False):
    """Rotary positions along time, height and width: `input` [N, L, H, D], each head's channels turned in pairs.

    `positions`: the grid (T, H, W) whose cells the tokens are, in that order (T * H * W == L), or a tensor [L, 3] or
    [N, L, 3] of real or whole positions (taken as float32; no gradient).  `axis_pairs`: how many pairs turn with each axis
    (default_axis_pairs); pair i of an axis turns by position * base^(-i / pairs of the axis) radians, channels behind the
    last pair pass.  Pair j of all is channels (2j, 2j + 1) with `interleaved`, else (j, j + all pairs).  Angles are exact to
    float32 for positions of up to 2^24 either way, and beyond off by 2^-48 turns a position."""
    if isinstance(input, torch.Tensor) and input.dim() == 4:
        pairs = default_axis_pairs(input.size(3)) if axis_pairs is None else axis_pairs
        real = isinstance(positions, torch.Tensor)
        out = _try_native("rotary3d", input, positions if real else None, (0, 0, 0) if real else positions, pairs, base, interleaved)
        if out is not None:
            return out
    _check_tensors("rotary3d", input=input)
    _check(input.dim() == 4, f"rotary3d: input must be [N, L, H, D], got {input.dim()} dimensions")
    N, L, H, D = input.shape
    _check(H > 0 and D > 0, "rotary3d: heads and their size must be positive")
    pairs = tuple(int(p) for p in (default_axis_pairs(D) if axis_pairs is None else axis_pairs))
    _check(len(pairs) == 3 and min(pairs) >= 0, f"rotary3d: axis_pairs must be three numbers of pairs, got {pairs}")
    _check(2 * sum(pairs) <= D, f"rotary3d: {sum(pairs)} pairs do not fit a head of {D} channels")
    grid = (0, 0, 0)
    if isinstance(positions, torch.Tensor):
        _check_tensors("rotary3d", input=input, positions=positions)
        _check(tuple(positions.shape) in ((L, 3), (N, L, 3)),
               f"rotary3d: positions must be [{L}, 3] or [{N}, {L}, 3], got {tuple(positions.shape)}")
        _check(not positions.requires_grad, "rotary3d: positions take no gradient")
        positions = positions.to(torch.float32).contiguous()
    else:
        grid, positions = tuple(int(v) for v in positions), None
        _check(len(grid) == 3 and min(grid) >= 0 and grid[0] * grid[1] * grid[2] == L,
               f"rotary3d: a grid of {grid} is not {L} tokens")
    if input.dtype == torch.float16:
        return rotary3d(input.float(), grid if positions is None else positions, pairs, base, interleaved).half()
    _check(input.dtype in _TYPES, f"rotary3d: unsupported dtype {input.dtype}")
    return _Rotary3dFunction.apply(input, positions, grid, pairs, float(base), bool(interleaved))


# ---------------------------------------------------------------- attention
def _inner_contiguous(t):
    return t if t.stride(3) == 1 or t.size(3) == 1 else t.contiguous()


def _part_workspace(desc, size, dev):
    """The workspace of a call, and its size: without room for partial sums where there is none."""
    nb = size(ctypes.byref(desc))
    try:
        return _workspace(nb, dev), nb
    except torch.cuda.OutOfMemoryError:
        desc.part_limit = -1
        nb = size(ctypes.byref(desc))
        return _workspace(nb, dev), nb


class _CrossAttentionFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value, key_lengths, key_mask, scale):
        lib, dev = _lib.load(), query.device
        q, k, v = (_inner_contiguous(t) for t in (query, key, value))
        N, Lq, Hq, D = q.shape
        Lk, Hkv = k.shape[1:3]
        desc = _lib.AttentionDesc(N, Lq, Lk, Hq, Hkv, D, _DT[q.dtype], scale, _long3(*q.stride()[:3]), _long3(*k.stride()[:3]),
                                  _long3(*v.stride()[:3]))
        out = torch.empty((N, Lq, Hq, D), dtype=q.dtype, device=dev)
        grad = any(ctx.needs_input_grad)
        lse = torch.empty((N, Hkv, Lq * (Hq // Hkv)), dtype=torch.float32, device=dev) if grad else None
        low = torch.empty_like(out) if grad and out.dtype == torch.bfloat16 else None
        with torch.cuda.device(dev):
            ws, nb = _part_workspace(desc, lib.d2c_attention_forward_workspace_bytes, dev)
            rc = lib.d2c_attention_forward(ctypes.byref(desc), _ptr(q), _ptr(k), _ptr(v), _ptr(key_lengths), _ptr(key_mask),
                                           _ptr(out), _ptr(low), _ptr(lse), _ptr(ws), nb, _stream(dev))
        _lib.check(rc, "cross_attention forward")
        ctx.save_for_backward(q, k, v, key_lengths, key_mask, out, low, lse)
        ctx.desc = desc
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        lib = _lib.load()
        q, k, v, key_lengths, key_mask, out, low, lse = ctx.saved_tensors
        desc, dev, need = ctx.desc, q.device, ctx.needs_input_grad
        desc.part_limit = 0
        q, k, v = (_inner_contiguous(t) for t in (q, k, v))
        desc.q_stride, desc.k_stride, desc.v_stride = (_long3(*t.stride()[:3]) for t in (q, k, v))
        g = grad_out.to(q.dtype).contiguous()
        gq, gk, gv = (torch.empty(t.shape, dtype=t.dtype, device=dev) if n else None for t, n in zip((q, k, v), need))
        with torch.cuda.device(dev):
            ws, nb = _part_workspace(desc, lib.d2c_attention_backward_workspace_bytes, dev)
            rc = lib.d2c_attention_backward(ctypes.byref(desc), _ptr(g), _ptr(q), _ptr(k), _ptr(v), _ptr(key_lengths),
                                            _ptr(key_mask), _ptr(out), _ptr(low), _ptr(lse), _ptr(gq), _ptr(gk), _ptr(gv),
                                            _ptr(ws), nb, _stream(dev))
        _lib.check(rc, "cross_attention backward")
        return gq, gk, gv, None, None, None


def cross_attention(query, key, value, key_lengths=None, key_mask=None, scale=None):
    """softmax(scale * query key^T) value, `query` [N, Lq, Hq, D], `key` and `value` [N, Lk, Hkv, D] with Hq a multiple of Hkv
    (query heads h * Hq / Hkv .. share key head h) and heads of up to 128 channels; `scale` 1 / sqrt(D) by default.

    `key_lengths` [N] (whole numbers, taken into 0 .. Lk): the first so many keys of a sample are there; `key_mask` [N, Lk]
    (bool): keys that may be read.  Keys and values that are not to be read have no influence whatever they hold (NaN
    included); a row without a key is 0 and has gradients of 0.  Any strides with the channels adjacent are read in place, a
    part of a wider projection for instance.  One row or thousands, one key or a long memory: where rows are few the work is
    split over the keys.  Sums in an order that sizes, strides and GPU alone determine, unless
    the GPU's memory has no room for the partial sums of split work (256 MB at most), which then is not split."""
    out = _try_native("cross_attention", query, key, value, key_lengths, key_mask, scale)
    if out is not None:
        return out
    _check_tensors("cross_attention", query=query, key=key, value=value, key_lengths=key_lengths, key_mask=key_mask)
    for name, t in (("query", query), ("key", key), ("value", value)):
        _check(t.dim() == 4, f"cross_attention: {name} must be [N, L, H, D], got {t.dim()} dimensions")
    N, Lq, Hq, D = query.shape
    _check(key.shape == value.shape, f"cross_attention: key {tuple(key.shape)} and value {tuple(value.shape)} differ in shape")
    _check(key.size(0) == N and key.size(3) == D,
           f"cross_attention: key {tuple(key.shape)} does not fit query {tuple(query.shape)}")
    Lk, Hkv = key.shape[1:3]
    _check(D > 0 and Hq > 0 and Hkv > 0 and Hq % Hkv == 0,
           f"cross_attention: {Hq} query heads must be a positive multiple of {Hkv} key heads, of {D} > 0 channels")
    _check(D <= 128, f"cross_attention: heads of up to 128 channels, got {D}")
    _check(query.dtype == key.dtype == value.dtype, "cross_attention: query, key and value must have one dtype")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    _check(0.0 < scale < math.inf, f"cross_attention: scale must be positive and finite, got {scale}")
    if key_lengths is not None:
        _check(tuple(key_lengths.shape) == (N,) and not key_lengths.is_floating_point() and not key_lengths.is_complex()
               and key_lengths.dtype != torch.bool, f"cross_attention: key_lengths must be {N} whole numbers")
        key_lengths = key_lengths.clamp(0, Lk) if key_lengths.dtype == torch.int64 else key_lengths
        key_lengths = key_lengths.to(torch.int32).contiguous()
    if key_mask is not None:
        _check(tuple(key_mask.shape) == (N, Lk) and key_mask.dtype == torch.bool,
               f"cross_attention: key_mask must be bool [{N}, {Lk}], got {key_mask.dtype} {tuple(key_mask.shape)}")
        key_mask = key_mask.contiguous()
    if query.dtype == torch.float16:
        return cross_attention(query.float(), key.float(), value.float(), key_lengths, key_mask, scale).half()
    _check(query.dtype in _TYPES, f"cross_attention: unsupported dtype {query.dtype}")
    return _CrossAttentionFunction.apply(query, key, value, key_lengths, key_mask, scale)


class LayerNorm(nn.LayerNorm):
    """`nn.LayerNorm` over the last dimension (parameters and state dict as there) on the kernels of this library."""

    def __init__(self, channels, eps=1e-5, elementwise_affine=True, bias=True, device=None, dtype=None):
        super().__init__(channels, eps, elementwise_affine, bias, device, dtype)
        if len(self.normalized_shape) != 1:
            raise ValueError("LayerNorm: one normalised dimension, the last")

    def forward(self, input):
        return layer_norm(input, self.weight, self.bias, self.eps)


class Memory(tuple):
    """(keys, values) of a feature map as `CrossAttention3d.remember` makes them, and the map's extents (T', H', W'), which
    masks of frames or cells are checked against."""

    def __new__(cls, key, value, dims):
        self = super().__new__(cls, (key, value))
        self.dims = tuple(dims)
        return self

    def __getnewargs__(self):      # (copies and pickles)
        return (*self, self.dims)


# (what walks over tuples of tensors, graphed callables for instance, walks over these, too)
register_pytree_node(Memory, lambda m: (list(m), m.dims), lambda pair, dims: Memory(*pair, dims))


class CrossAttention3d(nn.Module):
    """A clip's feature map reads the feature map of remembered frames, and adds what it read:

        x + out(attention(rotary(q(norm(x))), rotary(k(norm(memory))), v(norm(memory))))

    `channels` of the clip's map [N, channels, T, H, W], `memory_channels` (default: the same) of the memory's
    [N, memory_channels, T', H', W']; `heads` query heads over channels / heads channels each, `kv_heads` key heads.  `out` starts
    at zero, so that a network in which the block is new computes what it did (as the deformation branches of this package
    start)."""

    def __init__(self, channels, heads=8, kv_heads=None, memory_channels=None, bias=True, axis_pairs=None, base=10000.0,
                 eps=1e-5):
        super().__init__()
        memory_channels = channels if memory_channels is None else memory_channels
        kv_heads = heads if kv_heads is None else kv_heads
        if channels % heads or heads % kv_heads:
            raise ValueError(f"CrossAttention3d: {channels} channels, {heads} heads, {kv_heads} key heads do not divide")
        self.heads, self.kv_heads, self.head_channels = heads, kv_heads, channels // heads
        if self.head_channels > 128:
            raise ValueError(f"CrossAttention3d: heads of up to 128 channels, got {self.head_channels}")
        self.axis_pairs = tuple(default_axis_pairs(self.head_channels) if axis_pairs is None else axis_pairs)
        self.base = base
        self.norm = LayerNorm(channels, eps)
        self.memory_norm = LayerNorm(memory_channels, eps)
        self.query = nn.Linear(channels, channels, bias)
        self.key_value = nn.Linear(memory_channels, 2 * kv_heads * self.head_channels, bias)
        self.out = nn.Linear(channels, channels, bias)
        nn.init.zeros_(self.out.weight)
        if bias:
            nn.init.zeros_(self.out.bias)

    @staticmethod
    def _tokens(map):
        return map.flatten(2).transpose(1, 2)

    def _rotate(self, x, positions):
        return rotary3d(x, positions, self.axis_pairs, self.base)

    def remember(self, memory, positions=None):
        """Keys and values of `memory`, to be handed to any number of forward calls: the memory of a stream of frames is
        projected and turned once.  `positions` as rotary3d's; the memory's own grid by default.  A pair that knows the map's extents
        (Memory)."""
        N, _, *dims = memory.shape
        both = self.key_value(self.memory_norm(self._tokens(memory)))
        both = both.view(N, both.size(1), 2, self.kv_heads, self.head_channels)
        return Memory(self._rotate(both[:, :, 0], tuple(dims) if positions is None else positions), both[:, :, 1], dims)

    @staticmethod
    def _cells(mask, memory):
        """[N, cells] of a mask of frames or cells"""
        key, dims = memory[0], getattr(memory, "dims", None)
        cells = key.size(1)
        given = mask.flatten(1).size(1)
        if mask.dim() == 4 and given == cells and dims is not None:
            _check(tuple(mask.shape[1:]) == dims, f"CrossAttention3d: a mask of {tuple(mask.shape)} does not fit a memory of {dims}")
        mask = mask.flatten(1)
        # (of a pair that is no Memory the number of frames is not known: any that divides its cells)
        frames = dims is None and given > 0 and cells % given == 0 or dims is not None and given == dims[0]
        _check(given == cells or frames, f"CrossAttention3d: a mask of {given} does not fit {cells} cells"
               + ("" if dims is None else f" in {dims[0]} frames"))
        return mask if given == cells else mask.repeat_interleave(cells // given, 1)

    def forward(self, x, memory, positions=None, memory_positions=None, memory_lengths=None, memory_mask=None):
        """`memory`: a feature map, or what `remember` made of one.  `memory_lengths` [N]: how many of the memory's cells
        (frame after frame) are there; `memory_mask`: bool [N, T'] (frames) or [N, T', H', W'] or [N, cells]."""
        N, C, *dims = x.shape
        if not isinstance(memory, (tuple, list)):
            memory = self.remember(memory, memory_positions)
        key, value = memory
        if memory_mask is not None:
            memory_mask = self._cells(memory_mask, memory)
        q = self.query(self.norm(self._tokens(x)))
        q = q.view(N, q.size(1), self.heads, self.head_channels)
        q = self._rotate(q, tuple(dims) if positions is None else positions)
        read = cross_attention(q, key, value, memory_lengths, memory_mask)
        read = self.out(read.flatten(2))
        return x + read.transpose(1, 2).reshape(x.shape)
