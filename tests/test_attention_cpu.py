"""CPU checks of layer_norm, rotary3d, cross_attention and CrossAttention3d: the Python surface, what the C entry points refuse and
the workspaces that they ask for.  (No kernel is started here.)"""
import ctypes
import math

import pytest
import torch

import d2conv3d_amd as d2c
from d2conv3d_amd import _lib
from d2conv3d_amd.attention import default_axis_pairs

BF16 = 2


def _norm(**kw):
    d = dict(rows=10, x_stride=32, C=32, dtype=0, param_dtype=0, eps=1e-5)
    return _lib.LayerNormDesc(**{**d, **kw})


def _rotary(pairs=(4, 6, 6), grid=(2, 3, 4), x_stride=(24 * 128, 128, 32), **kw):
    d = dict(N=1, L=24, H=4, D=32, interleaved=0, direction=1, dtype=0, base=1e4, position_stride=0)
    i3, l3 = ctypes.c_int32 * 3, ctypes.c_int64 * 3
    return _lib.Rotary3dDesc(pairs=i3(*pairs), grid=i3(*grid), x_stride=l3(*x_stride), **{**d, **kw})


def _attention(**kw):
    d = {**dict(N=1, Lq=100, Lk=200, Hq=4, Hkv=2, D=32, dtype=0, scale=0.1), **kw}
    l3 = ctypes.c_int64 * 3
    q, k = (l3(d[n] * d[h] * d["D"], d[h] * d["D"], d["D"]) for n, h in (("Lq", "Hq"), ("Lk", "Hkv")))
    return _lib.AttentionDesc(q_stride=q, k_stride=k, v_stride=k, **d)


def _call(fn, desc, pointers):
    return getattr(_lib.load(), fn)(None if desc is None else ctypes.byref(desc), *pointers)


@pytest.mark.parametrize("desc,text", [
    (None, "null description"), (_norm(rows=-1), "must not be negative"), (_norm(C=0), "positive"), (_norm(dtype=1), "float32 or bfloat16"),
    (_norm(param_dtype=BF16), "parameters"), (_norm(C=1 << 20), "up to"), (_norm(eps=math.nan), "eps"), (_norm(), "null tensor")])
def test_layer_norm_refuses(desc, text):
    assert _call("d2c_layer_norm_forward", desc, [None] * 6) != 0 and text in _lib.last_error()
    assert _call("d2c_layer_norm_backward", desc, [None] * 8 + [0, None]) != 0 and text in _lib.last_error()


@pytest.mark.parametrize("desc,text", [
    (None, "null description"), (_rotary(dtype=1), "float32 or bfloat16"), (_rotary(N=-1), "negative"), (_rotary(H=0), "positive"),
    (_rotary(N=1 << 17), "too many samples"), (_rotary(pairs=(8, 8, 1)), "do not fit"), (_rotary(pairs=(-1, 2, 2)), "out of range"),
    (_rotary(direction=0), "direction"), (_rotary(base=0.0), "base"), (_rotary(base=math.inf), "base"), (_rotary(), "null tensor")])
def test_rotary_refuses(desc, text):
    assert _call("d2c_rotary3d", desc, [None] * 4) != 0 and text in _lib.last_error()


def test_rotary_refuses_a_grid_of_another_number():
    assert _call("d2c_rotary3d", _rotary(grid=(2, 3, 5)), [256, None, 256, None]) != 0 and "tokens" in _lib.last_error()


@pytest.mark.parametrize("desc,text", [
    (None, "null description"), (_attention(dtype=1), "float32 or bfloat16"), (_attention(Lk=-1), "negative"), (_attention(D=0), "positive"),
    (_attention(Hq=3), "no multiple"), (_attention(D=129), "up to 128"), (_attention(scale=0.0), "scale"),
    (_attention(scale=math.inf), "scale"), (_attention(scale=math.nan), "scale"), (_attention(Lk=1 << 30), "too many"),
    (_attention(Lq=1 << 30), "too many"), (_attention(N=1 << 24), "too many"), (_attention(), "null tensor")])
def test_attention_refuses(desc, text):
    assert _call("d2c_attention_forward", desc, [None] * 9 + [0, None]) != 0 and text in _lib.last_error()
    assert _call("d2c_attention_backward", desc, [None] * 13 + [0, None]) != 0 and text in _lib.last_error()


def test_sizes_of_nothing_are_no_error():
    for desc in (_attention(N=0), _attention(Lq=0)):
        assert _call("d2c_attention_forward", desc, [None] * 9 + [0, None]) == 0
        assert _lib.load().d2c_attention_forward_workspace_bytes(ctypes.byref(desc)) == 0
    assert _call("d2c_rotary3d", _rotary(L=0, grid=(0, 3, 4)), [None] * 4) == 0
    assert _call("d2c_layer_norm_forward", _norm(rows=0), [None] * 6) == 0


def test_workspaces_are_asked_for_and_checked():
    lib = _lib.load()
    for dtype in (0, BF16):
        desc = _attention(Lq=16, Lk=30000, Hkv=1, dtype=dtype)        # one walk (whatever the GPU): shared, and partial sums need room
        need = lib.d2c_attention_forward_workspace_bytes(ctypes.byref(desc))
        assert need > 0 and need % 256 == 0
        for ws, size in ((None, need), (256, need - 1), (256 + 8, need)):
            assert _call("d2c_attention_forward", desc, [256, 256, 256, None, None, 256, None, None, ws, size, None]) != 0
            assert "workspace" in _lib.last_error()
        need = lib.d2c_attention_backward_workspace_bytes(ctypes.byref(desc))
        assert need >= 16 * 4 * 4
        assert _call("d2c_attention_backward", desc, [256] * 4 + [None, None, 256, None, 256, 256, 256, 256, 256, need - 1, None]) != 0
        assert "workspace" in _lib.last_error()
    assert lib.d2c_attention_forward_workspace_bytes(ctypes.byref(_attention(D=129))) == 0
    assert lib.d2c_layer_norm_backward_workspace_bytes(ctypes.byref(_norm(rows=5000, x_stride=32))) >= 2 * 32 * 4


def test_no_path_on_the_cpu():
    x = torch.randn(2, 6, 4, 32)
    with pytest.raises(RuntimeError, match="on the GPU"):
        d2c.layer_norm(x)
    with pytest.raises(RuntimeError, match="on the GPU"):
        d2c.rotary3d(x, (1, 2, 3))
    with pytest.raises(RuntimeError, match="on the GPU"):
        d2c.cross_attention(x, x, x)
    with pytest.raises(RuntimeError, match="must be a Tensor"):
        d2c.cross_attention(x.tolist(), x, x)


def test_the_block_is_a_module_like_others():
    block = d2c.CrossAttention3d(64, heads=4, kv_heads=2, memory_channels=48)
    names = {n: tuple(p.shape) for n, p in block.named_parameters()}
    assert names["query.weight"] == (64, 64) and names["key_value.weight"] == (64, 48) and names["memory_norm.weight"] == (48,)
    assert not bool(block.out.weight.any())
    norm = d2c.LayerNorm(48)
    norm.load_state_dict(torch.nn.LayerNorm(48).state_dict())
    for args in (dict(channels=65, heads=4), dict(channels=64, heads=4, kv_heads=3), dict(channels=1040, heads=8)):
        with pytest.raises(ValueError):
            d2c.CrossAttention3d(**args)
    with pytest.raises(ValueError):
        d2c.LayerNorm((4, 8))


@pytest.mark.parametrize("D", [2, 6, 24, 33, 64, 80, 128])
def test_default_pairs_fill_the_head(D):
    pairs = default_axis_pairs(D)
    assert sum(pairs) == D // 2 and min(pairs) >= 0 and pairs[1] == pairs[2]
