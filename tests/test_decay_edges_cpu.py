"""The decay-attention layer's refusals and autograd rules, without a GPU."""
import ctypes

import pytest
import torch


# ------------------------------------------------------------------------------------------ states in order
@pytest.mark.parametrize("src,dst,n_rows,n_src", [
    ((4096, 8192), (8192, 4096), 4, 4),          # two states that would change places
    ((4096, 8192), (16384, 4096 + 64), 4, 4),    # a part of another state
    ((4096, 8192), (16384, 16384 + 128), 4, 4),  # two outputs over one another
    ((4096, 8192), (16384, 8192), 2, 4),
    ((4096, 8192), (16384, (1 << 20) - 64), 4, 4),   # the order itself
])
def test_reorder_refuses_outputs_over_any_state_and_one_another(src, dst, n_rows, n_src):
    from icml_b200 import _lib
    arr = ctypes.c_void_p * 2
    rc = _lib.lib().pgf_beam_reorder(arr(*src), arr(*dst), (ctypes.c_int64 * 2)(64, 64), 2, 1 << 20, n_rows, n_src, None)
    assert rc != 0 and "overwrite" in _lib.last_error()
