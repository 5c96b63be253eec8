"""layer_norm where every workgroup takes several rows: forward launches have up to 16 workgroups to a compute unit of 1 to 32 rows each, backward ones 4, and
walk over what is behind.  Definition and bounds: test_gpu_layer_norm.py; computed on the GPU in float64, as the inputs are large."""
import pytest
import torch

import d2conv3d_amd as d2c
from test_gpu_layer_norm import make, reference

pytestmark = pytest.mark.gpu


# channels, and the rows that a workgroup takes at once, for both types (a row is 16-byte vectors on 8 to 256 lanes)
@pytest.mark.parametrize("C,types,per", [
    (16, (torch.float32, torch.float32), 32), (60, (torch.bfloat16, torch.float32), 32), (64, (torch.float32, torch.float32), 16),
    (128, (torch.bfloat16, torch.bfloat16), 16), (128, (torch.float32, torch.float32), 8), (250, (torch.bfloat16, torch.float32), 8),
    (256, (torch.float32, torch.float32), 4), (512, (torch.bfloat16, torch.float32), 4), (500, (torch.float32, torch.float32), 4),
    (1000, (torch.bfloat16, torch.bfloat16), 4), (2100, (torch.float32, torch.float32), 1), (2100, (torch.bfloat16, torch.float32), 1),
    (8200, (torch.bfloat16, torch.float32), 1), (8200, (torch.float32, torch.float32), 1)])
def test_several_rows_to_a_workgroup(C, types, per, dev):
    cus = torch.cuda.get_device_properties(dev).multi_processor_count
    rows = 16 * cus * per + 4 * cus * per // 3 + 1       # (forward: a second row for some; backward: five or six)
    print("layer_norm", rows, C, types, flush=True)
    x, w, b, g = (t.to(dev) for t in make((rows, C), *types, seed=C))
    want, bounds = reference(x, w, b, g)
    args = [t.requires_grad_() for t in (x, w, b)]
    out = d2c.layer_norm(*args)
    got = (out, *torch.autograd.grad(out, args, g))
    for name, a, e, bound in zip(("out", "grad_input", "grad_weight", "grad_bias"), got, want, bounds):
        over = (a.detach().double() - e).abs() / (1.05 * bound + 1e-30)
        assert not bool((~(over <= 1.0)).any()), f"{name}: worst {over.max().item():.2f} of the bound, NaN {int(a.isnan().sum())}"
