"""What the gated feed-forward block and rotary positions refuse, decided on the host: no GPU, no launch."""
import ctypes
import math

import pytest
import torch

import matterformer_b200 as mfb
from matterformer_b200 import _lib
from matterformer_b200.rotary import RotaryPositions, rotate_torch
from matterformer_b200.trunk import EDMModel, GatedMlp, RegularAttention, TransformerTrunk

OK, OFF = 0x7F0000001000, 0x7F0000001002  # fake device addresses: validation never dereferences them


def _mlp(**over):
    a = _lib.MfGatedMlpArgs(rows=4, dim=16, hidden=24, dim_out=16, dtype=_lib.MF_DTYPE_BF16, grad_dtype=_lib.MF_DTYPE_BF16, x=OK, w_in=OK, w_out=OK, act=OK,
                            y=OK, pre=OK, grad_y=OK)  # fmt: skip
    for name, value in over.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("over,message", [
    ({"dtype": _lib.MF_DTYPE_F32}, "only supports float16/bfloat16"), ({"grad_dtype": _lib.MF_DTYPE_F16}, "weight gradients come in"),
    ({"activation": 2}, "unknown activation"), ({"activation": -1}, "unknown activation"), ({"rows": -1}, "rows must lie"),
    ({"rows": 2**31}, "rows must lie"), ({"dim": 12}, "multiples of 8"), ({"hidden": 0}, "multiples of 8"), ({"dim_out": -8}, "multiples of 8"),
    ({"dim": 2**30}, "above 2"), ({"x": None}, "null tensor"), ({"w_in": None}, "null tensor"), ({"act": None}, "null tensor"),
    ({"x": OFF}, "16-byte aligned"), ({"b_in": OFF}, "16-byte aligned"), ({"grad_x": OFF}, "16-byte aligned"),
])  # fmt: skip
def test_gated_mlp_arguments(over, message):
    L = _lib.lib()
    for fn in (L.mf_gated_mlp_fwd, L.mf_gated_mlp_bwd):
        assert fn(ctypes.byref(_mlp(**over)), None) == _lib.MF_ERR_INVALID_ARGUMENT
        assert message in _lib.last_error()


def test_gated_mlp_more_arguments():
    L = _lib.lib()
    assert L.mf_gated_mlp_fwd(None, None) == L.mf_gated_mlp_bwd(None, None) == _lib.MF_ERR_INVALID_ARGUMENT
    assert L.mf_gated_mlp_fwd(ctypes.byref(_mlp(y=None)), None) == _lib.MF_ERR_INVALID_ARGUMENT
    for name in ("pre", "grad_y"):
        assert L.mf_gated_mlp_bwd(ctypes.byref(_mlp(**{name: None})), None) == _lib.MF_ERR_INVALID_ARGUMENT
    assert L.mf_gated_mlp_bwd(ctypes.byref(_mlp(grad_x=OK)), None) == _lib.MF_ERR_WORKSPACE_TOO_SMALL
    need = L.mf_gated_mlp_bwd_workspace_bytes(ctypes.byref(_mlp(grad_x=OK)))
    assert L.mf_gated_mlp_bwd(ctypes.byref(_mlp(grad_x=OK, workspace=OK, workspace_bytes=need - 1)), None) == _lib.MF_ERR_WORKSPACE_TOO_SMALL
    assert need >= 4 * 48 * 2
    assert L.mf_gated_mlp_bwd_workspace_bytes(ctypes.byref(_mlp(rows=0))) == L.mf_gated_mlp_bwd_workspace_bytes(None) == 0
    assert L.mf_gated_mlp_fwd(ctypes.byref(_mlp(rows=0, x=None)), None) == _lib.MF_OK  # nothing to do
    assert L.mf_gated_mlp_status(None, None) == _lib.MF_ERR_INVALID_ARGUMENT
    status = ctypes.c_int32(0)
    for kind, limit in ((4, 1000), (-1, 1000), (0, 0), (0, 2**31 + 1)):
        assert L.mf_selftest_gated_mlp_give_up(ctypes.byref(_mlp()), 0, kind, limit, ctypes.byref(status), None) == _lib.MF_ERR_INVALID_ARGUMENT


def _rotary(**over):
    table = (ctypes.c_double * 200)(*([1.0] * 200))
    a = _lib.MfRotaryArgs(batch=2, tokens=3, head_dim=16, axes=1, pairs=8, dtype=_lib.MF_DTYPE_BF16, tensors=1, positions=OK)
    a.frequencies = ctypes.cast(table, ctypes.POINTER(ctypes.c_double))
    t = a.tensor[0]
    t.input = t.out = OK
    t.heads, t.rotates = 2, 1
    for name, value in over.items():
        setattr(t if hasattr(t, name) else a, name, value)
    a.keep = table
    return a


@pytest.mark.parametrize("over,message", [
    ({"dtype": 3}, "only supports"), ({"batch": -1}, "negative size"), ({"head_dim": 0}, "negative size"), ({"pairs": 9}, "need a head_dim"),
    ({"pairs": 0}, "must lie in"), ({"axes": 0}, "must lie in"), ({"pairs": 129, "head_dim": 512}, "must lie in"), ({"axes": 2**20, "pairs": 2**12}, "must lie in"),
    ({"layout": 2}, "unknown layout"), ({"position_type": 4}, "unknown position type"), ({"tensors": 0}, "between one and three"), ({"tensors": 4}, "between one and three"),
    ({"frequencies": ctypes.POINTER(ctypes.c_double)()}, "null frequencies"), ({"heads": -1}, "negative size"), ({"input": None}, "null tensor"),
    ({"out": None}, "null tensor"), ({"input": OK + 1}, "unaligned"), ({"positions": None}, "null positions"),
])  # fmt: skip
def test_rotary_arguments(over, message):
    assert _lib.lib().mf_rotary(ctypes.byref(_rotary(**over)), None) == _lib.MF_ERR_INVALID_ARGUMENT
    assert message in _lib.last_error()


def test_rotary_elements_a_token():
    assert _lib.lib().mf_rotary(ctypes.byref(_rotary(heads=2**23 + 1)), None) == _lib.MF_ERR_INVALID_ARGUMENT
    assert "more than 2^27 elements a token" in _lib.last_error()


def test_rotary_nothing_to_do():
    L = _lib.lib()
    assert L.mf_rotary(None, None) == _lib.MF_ERR_INVALID_ARGUMENT
    for over in ({"batch": 0}, {"tokens": 0}, {"heads": 0}):
        assert L.mf_rotary(ctypes.byref(_rotary(positions=None, **over)), None) == _lib.MF_OK


def test_frequencies():
    plain = mfb.rotary_frequencies(8)
    assert plain.dtype == torch.float64 and torch.allclose(plain, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)
    assert torch.equal(mfb.rotary_frequencies(8, scaling="linear", factor=4.0), plain / 4)
    ntk = mfb.rotary_frequencies(8, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], plain[-1] / 4, rel_tol=1e-14)
    parts = mfb.rotary_frequencies(8, scaling="parts", factor=4.0, original_length=2000.0)
    turns = 2000.0 * plain / (2 * math.pi)  # 318, 31.8, 3.18, 0.318
    assert parts[0] == plain[0] and math.isclose(parts[3], plain[3] / 4, rel_tol=1e-15)
    for p in (1, 2):
        kept = (turns[p].item() - 1) / 31
        assert math.isclose(parts[p], plain[p] * (kept + (1 - kept) / 4), rel_tol=1e-14)
    assert mfb.rotary_frequencies(12, axes=3).shape == (3, 2)
    for bad in ({"rotary_dim": 7}, {"rotary_dim": 0}, {"rotary_dim": 8, "axes": 3}, {"rotary_dim": 8, "base": 0.0}, {"rotary_dim": 8, "factor": -1.0},
                {"rotary_dim": 8, "scaling": "half"}, {"rotary_dim": 8, "scaling": "parts"}, {"rotary_dim": 8, "scaling": "parts", "original_length": 5.0, "slow": 9.0, "fast": 3.0}):  # fmt: skip
        with pytest.raises(ValueError):
            mfb.rotary_frequencies(**bad)


def test_frequencies_stay_on_the_host():
    with torch.device("meta"):
        assert mfb.rotary_frequencies(8).device.type == mfb.RotaryPositions(8).frequencies.device.type == "cpu"


def test_python_layer():
    x, w, v = torch.zeros(4, 16), torch.zeros(48, 16), torch.zeros(16, 24)
    with pytest.raises(RuntimeError, match="requires CUDA tensors"):
        mfb.gated_mlp(x, w, v)
    table = mfb.rotary_frequencies(8)
    with pytest.raises(RuntimeError, match="requires CUDA tensors"):
        mfb.rotary_embedding(torch.zeros(1, 1, 2, 8), None, torch.arange(2), table)
    with pytest.raises(RuntimeError, match="requires CUDA tensors"):
        mfb.rotary_packed(torch.zeros(1, 2, 24), 1, torch.arange(2), table)
    with pytest.raises(ValueError, match="expected"):
        mfb.rotary_packed(torch.zeros(1, 2, 24), 5, torch.arange(2), table)
    with pytest.raises(ValueError, match="expected"):
        mfb.rotary_embedding(torch.zeros(1, 2, 8), None, torch.arange(2), table)
    with pytest.raises(ValueError, match="expected"):
        mfb.rotary_embedding(torch.zeros(1, 1, 2, 8), torch.zeros(1, 1, 3, 8), torch.arange(2), table)


def test_modules():
    rotary = RotaryPositions(rotary_dim=6, axes=3, base=50.0)
    assert rotary.frequencies.shape == (3, 1) and rotary.frequencies is rotary.frequencies
    with pytest.raises(ValueError, match="above the head size"):
        RegularAttention(32, 8, rotary=rotary)
    with pytest.raises(ValueError, match="needs `positions`"):
        RegularAttention(32, 4, rotary=rotary)(torch.zeros(1, 3, 32))
    with pytest.raises(ValueError, match="are for a layer"):
        RegularAttention(32, 4)(torch.zeros(1, 3, 32), positions=torch.zeros(1, 3, 3))
    with pytest.raises(ValueError, match="needs `positions`"):
        TransformerTrunk(32, 4, ["mha"], rotary=rotary)(torch.zeros(1, 3, 32), torch.zeros(1, 32))
    with pytest.raises(ValueError, match="3 axes"):
        EDMModel(d_model=32, n_heads=4, n_layers=1, rotary=RotaryPositions(rotary_dim=4))
    with pytest.raises(ValueError, match="Unsupported activation"):
        GatedMlp(32, activation="relu")
    with pytest.raises(ValueError, match="Unsupported mlp_type"):
        TransformerTrunk(32, 4, ["mha"], mlp_type="wide")
    assert GatedMlp(512).hidden == 1368 and GatedMlp(64, hidden=40).fc1.weight.shape == (80, 64)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_attention_with_positions_on_the_cpu(layout):
    """Scores depend on differences of positions alone, and the layer without a turn is the plain one."""
    torch.manual_seed(0)
    layer = RegularAttention(32, 4, rotary=RotaryPositions(rotary_dim=6, axes=3, base=50.0, layout=layout)).double()
    x, pos = torch.randn(2, 7, 32, dtype=torch.float64), torch.randn(2, 7, 3, dtype=torch.float64)
    pad = torch.zeros(2, 7, dtype=torch.bool)
    pad[1, 5:] = True
    y = layer(x, key_padding_mask=pad, positions=pos)
    moved = layer(x, key_padding_mask=pad, positions=pos + torch.tensor([3.0, -1.0, 0.5]))
    torch.testing.assert_close(moved, y, rtol=1e-9, atol=1e-9)
    plain = RegularAttention(32, 4).double()
    plain.load_state_dict(layer.state_dict())
    still = layer(x, key_padding_mask=pad, positions=torch.zeros_like(pos))
    torch.testing.assert_close(still[0], plain(x, key_padding_mask=pad)[0], rtol=1e-9, atol=1e-9)
    torch.testing.assert_close(still[1, :5], plain(x, key_padding_mask=pad)[1, :5], rtol=1e-9, atol=1e-9)
    assert (y - still).abs().max() > 1e-3
    z = rotate_torch(torch.ones(1, 1, 1, 8), torch.tensor([1.0]), mfb.rotary_frequencies(4), layout, amplitude=2.0)
    assert z.shape == (1, 1, 1, 8) and torch.equal(z[..., 4:], torch.ones(1, 1, 1, 4))


def test_gated_trunk_on_the_cpu():
    """Runs, and its parameters get gradients that differences confirm."""
    torch.manual_seed(1)
    trunk = TransformerTrunk(16, 2, ["mha", "simplicial"], mlp_type="gated", simplicial_impl="torch", rotary=RotaryPositions(rotary_dim=6, axes=3)).double()
    for p in trunk.parameters():
        torch.nn.init.normal_(p, std=0.3)
    x, cond, pos = (torch.randn(*s, dtype=torch.float64) for s in ((2, 5, 16), (2, 16), (2, 5, 3)))
    pad = torch.zeros(2, 5, dtype=torch.bool)
    pad[1, 3:] = True

    def loss():
        return trunk(x, cond, pad_mask=pad, positions=pos).square().sum()

    grads = torch.autograd.grad(loss(), list(trunk.parameters()))
    v = [torch.randn_like(p) for p in trunk.parameters()]
    with torch.no_grad():
        values = []
        for h in (1e-5, -1e-5):
            for p, d in zip(trunk.parameters(), v):
                p.add_(h * d)
            values.append(loss().item())
            for p, d in zip(trunk.parameters(), v):
                p.sub_(h * d)
    slope = sum((g * d).sum().item() for g, d in zip(grads, v))
    assert math.isclose((values[0] - values[1]) / 2e-5, slope, rel_tol=1e-4)
