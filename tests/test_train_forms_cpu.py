"""CPU tests of the forms in which tensors may reach the training entry points."""

import ctypes

import pytest

from flash_mlm import _lib
from test_train_cpu import bwd_args


@pytest.mark.parametrize("layout,batch", [(_lib.FMLM_BWD_PACKED, 1), (_lib.FMLM_BWD_DENSE, 2)])
def test_the_stride_of_a_single_row_is_free(layout, batch):
    """One row per head, in a projection's strides: the next check (of the workspace) is reached."""
    def view(heads):  # [B, 1, H, D] transposed
        return _lib.View4(1 << 20, 1, heads, batch, 64 * heads, 64, 64 * heads)

    a = bwd_args(layout=layout, total_q_len=1, seq_len=1, q=view(4), dout=view(4), k=view(2), v=view(2), workspace=None)
    L = _lib.lib()
    assert L.fmlm_attn_bwd(ctypes.byref(a), None) == -1
    assert "workspace" in L.fmlm_last_error().decode()
    a.dout = _lib.View4(1 << 20, 1, 4, batch, 64, 128, 512)  # heads apart
    assert L.fmlm_attn_bwd(ctypes.byref(a), None) == -1
    assert "contiguous" in L.fmlm_last_error().decode()
