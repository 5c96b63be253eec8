"""cross_attention of up to 8 rows of a key head, bfloat16: the weights are held in float32, so that the output before it is rounded (output + low) is off by
float32 arithmetic alone: E = 2 u32 (D + 64 + keys / 8 + 4 max_s) sum_j p_j |v_j|, as test_gpu_attention.py has it, and 2^-16 |o| for low's own rounding."""
import math

import pytest
import torch

import d2conv3d_amd as d2c
from d2conv3d_amd import attention
from test_gpu_attention import make, make_masks

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [7, 24, 40, 64, 80, 128])
@pytest.mark.parametrize("N,Lq,Lk,Hq,Hkv,kind", [(2, 1, 700, 2, 2, "none"), (3, 1, 5000, 4, 2, "both"), (1, 4, 333, 2, 2, "mask"), (1, 4, 900, 4, 2, "none"),
                                                 (2, 8, 3000, 1, 1, "lengths"), (2, 1, 50, 4, 4, "none")])
def test_float32_weights(N, Lq, Lk, Hq, Hkv, kind, D, dev, monkeypatch):
    monkeypatch.setattr(attention, "_try_native", lambda *a: None)      # (whose node shows what it kept)
    q, k, v, _ = make(N, Lq, Lk, Hq, Hkv, D, torch.bfloat16, D + Lk, std=1.5)
    lengths, mask = make_masks(kind, N, Lk, 3)
    ok = torch.ones(N, Lk, dtype=torch.bool)
    if lengths is not None:
        ok &= torch.arange(Lk) < lengths[:, None]
    if mask is not None:
        ok &= mask
    rep = Hq // Hkv
    Q = q.double().permute(0, 2, 1, 3)
    K, V = (t.double().permute(0, 2, 1, 3).repeat_interleave(rep, 1) for t in (k, v))
    s = Q @ K.transpose(-1, -2).contiguous() / math.sqrt(D)
    smax = (Q.abs() @ K.abs().transpose(-1, -2).contiguous()).max().item() / math.sqrt(D)
    p = torch.where(ok[:, None, None], s, -math.inf).softmax(-1).nan_to_num(0.0)
    want, A = (p @ V).permute(0, 2, 1, 3), (p @ V.abs()).permute(0, 2, 1, 3)
    bound = 2 * 2.0 ** -24 * (D + 64 + Lk / 8 + 4 * smax) * A + 2.0 ** -16 * want.abs()
    out = d2c.cross_attention(q.to(dev).requires_grad_(), k.to(dev), v.to(dev), None if lengths is None else lengths.to(dev),
                              None if mask is None else mask.to(dev))
    got = (out.detach().double() + out.grad_fn.saved_tensors[6].double()).cpu()
    over = (got - want).abs() / (1.05 * bound + 1e-30)
    assert not bool((~(over <= 1.0)).any()), f"worst {over.max().item():.2f} of the bound"
