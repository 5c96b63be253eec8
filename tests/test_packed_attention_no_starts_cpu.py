"""packed_attention's C interface wants starts whenever there are tokens, also where there are no sequences: the kernels read the first of them."""
import ctypes

import pytest

from d2conv3d_amd import _lib
from test_packed_attention_cpu import desc


@pytest.mark.parametrize("sequences", [0, 1, 3])
@pytest.mark.parametrize("tokens", [dict(queries=100, keys=100), dict(queries=100, keys=0), dict(queries=0, keys=100)])
@pytest.mark.parametrize("key_starts", [None, 4096])
def test_no_starts(sequences, tokens, key_starts):
    lib = _lib.load()
    q = ctypes.byref(desc(sequences=sequences, **tokens))
    some, other = ctypes.c_void_p(4096), ctypes.c_void_p(key_starts)
    # (a workspace that is too small: a call whose starts are not missed ends there, and launches nothing)
    if tokens["queries"]:
        assert lib.d2c_packed_attention_forward(q, some, some, some, None, other, some, None, some, None, 0, None) != 0 and "null" in _lib.last_error()
    assert lib.d2c_packed_attention_backward(q, *(some,) * 4, None, other, *(some,) * 6, None, 0, None) != 0 and "null" in _lib.last_error()
