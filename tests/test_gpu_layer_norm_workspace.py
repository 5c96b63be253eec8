"""The workgroups' sums of layer norm's parameters: how much room they take at most."""
import ctypes

import pytest
import torch

from d2conv3d_amd import _lib

pytestmark = pytest.mark.gpu


def test_room_for_the_workgroups_sums(dev):
    need = _lib.load().d2c_layer_norm_backward_workspace_bytes
    for C in (1, 16, 257, 1024, 2048, 4100, 8192, 16383, 16384):
        for dtype, params in ((0, 0), (2, 0), (2, 2)):
            for rows in (0, 1, 1000, 100000, 1 << 30):
                q = _lib.LayerNormDesc(rows=rows, x_stride=C, C=C, dtype=dtype, param_dtype=params, eps=1e-5)
                assert 2 * C * 4 <= need(ctypes.byref(q)) <= (64 << 20), (rows, C)
