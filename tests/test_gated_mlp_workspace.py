"""What the gated block's backward pass asks for as workspace: what the wanted gradients need."""
import ctypes

import pytest

from matterformer_b200 import _lib

OK = 0x7F0000001000  # a fake device address: sizes never dereference it


def _bytes(rows, **wanted):
    a = _lib.MfGatedMlpArgs(rows=rows, dim=512, hidden=1368, dim_out=512, dtype=_lib.MF_DTYPE_BF16, grad_dtype=_lib.MF_DTYPE_BF16)
    for name in wanted:
        setattr(a, "grad_" + name, OK)
    return _lib.lib().mf_gated_mlp_bwd_workspace_bytes(ctypes.byref(a))


@pytest.mark.parametrize("rows", [1, 5000, 100_000])
def test_the_gradient_of_the_pre_activations_only_where_it_is_formed(rows):
    formed = rows * 2 * 1368 * 2
    for name in ("x", "w_in", "b_in"):
        assert _bytes(rows, **{name: True}) >= formed
    assert _bytes(rows) == 0
    assert _bytes(rows, b_out=True) == 296 * 512 * 4
    with_x, without = _bytes(rows, x=True, w_out=True), _bytes(rows, w_out=True)
    assert with_x - without == -(-formed // 256) * 256
