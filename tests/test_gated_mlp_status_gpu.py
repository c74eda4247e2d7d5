"""The status of expired waits of the gated block: told once, to the next who asks."""
import ctypes

import pytest
import torch

import matterformer_b200 as mfb
from matterformer_b200 import _lib, gated

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _expire(host_status=None):
    """A call whose waits expire; without `host_status` it leaves its status where every call does."""
    g = torch.Generator().manual_seed(0)
    ops = [(torch.randn(*s, generator=g) * 0.1).to(BF16).cuda() for s in ((600, 64), (2 * 648, 64), (520, 648))]
    a = gated._args(*ops, None, None, "silu", BF16)
    act, y = torch.empty(600, 648, dtype=BF16, device="cuda"), torch.empty(600, 520, dtype=BF16, device="cuda")
    a.act, a.y = act.data_ptr(), y.data_ptr()
    _lib.launch(_lib.lib().mf_selftest_gated_mlp_give_up, y.device, ctypes.byref(a), 0, 0, 40000, host_status)
    torch.cuda.synchronize()
    return ops


def test_reported_once():
    assert mfb.gated_mlp_status() == 0
    ops = _expire()
    assert mfb.gated_mlp_status() == _lib.MF_ERR_DEVICE_TIMEOUT
    assert mfb.gated_mlp_status() == 0
    mfb.gated_mlp(*ops)
    assert mfb.gated_mlp_status() == 0


def test_the_self_test_keeps_its_status_to_itself():
    _expire()
    status = ctypes.c_int32(0)
    _expire(ctypes.byref(status))
    assert status.value == _lib.MF_ERR_DEVICE_TIMEOUT
    assert mfb.gated_mlp_status() == _lib.MF_ERR_DEVICE_TIMEOUT  # of the first call, not erased by the second


@pytest.mark.parametrize("wide", [False, True])
def test_checked_calls_raise(wide):
    """With the check on, forward and backward pass raise for a wait that expired since the last look."""
    previous = mfb.set_check_status(True)
    try:
        ops = _expire()
        leaves = [ops[0].requires_grad_(), *(t.float() if wide else t for t in ops[1:])]
        with pytest.raises(RuntimeError, match="device-side wait"):
            mfb.gated_mlp(*leaves)
        y = mfb.gated_mlp(*leaves)
        _expire()
        with pytest.raises(RuntimeError, match="device-side wait"):
            torch.autograd.grad(y, leaves[0], torch.ones_like(y), retain_graph=True)
        torch.autograd.grad(y, leaves[0], torch.ones_like(y))
    finally:
        mfb.set_check_status(previous)
    assert mfb.gated_mlp_status() == 0
