"""Positions as models have them: coordinates with a gradient, of 16 bits, not a number on padded tokens; layers of an earlier version."""
import copy
import pickle

import pytest
import torch

import matterformer_b200 as mfb
from matterformer_b200.rotary import RotaryPositions, rotate_torch
from matterformer_b200.trunk import EDMModel, RegularAttention, TransformerTrunk

ROTARY = RotaryPositions(rotary_dim=24, axes=3, base=50.0)


def _layer():
    torch.manual_seed(0)
    return RegularAttention(128, 4, rotary=ROTARY)


def _inputs(B=3, N=20):
    g = torch.Generator().manual_seed(1)
    pad = torch.arange(N)[None, :] >= torch.tensor([N, N // 2, 3])[:B, None]
    return torch.randn(B, N, 128, generator=g), torch.randn(B, N, 3, generator=g), pad, torch.randn(B, N, 128, generator=g).masked_fill(pad[..., None], 0.0)


def _off(a, b):
    return ((a.double().cpu() - b.double().cpu()).norm() / b.double().norm()).item()


@pytest.mark.gpu
@pytest.mark.parametrize("scattered", [False, True])  # padding in front: the dense core
def test_coordinates_with_a_gradient(scattered):
    """On CUDA as on the CPU; in bf16 some ten roundings of 2^-9 on the way to scores and back, twice as many in a gradient: 3 %."""
    layer, (x, pos, pad, dy) = _layer(), _inputs()
    if scattered:
        pad, dy = pad.flip(1), dy.flip(1)

    def run(layer, device, dtype, low):
        p = pos.to(device, dtype).requires_grad_()
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=low):
            y = layer(x.to(device, dtype), key_padding_mask=pad.to(device), positions=p)
        y = y.masked_fill(pad.to(device)[..., None], 0.0)
        return y.detach(), torch.autograd.grad(y, p, dy.to(device, y.dtype))[0]

    want = run(copy.deepcopy(layer).double(), "cpu", torch.float64, False)
    assert want[1].abs().max() > 1e-3
    layer = layer.cuda()
    for low, bound in ((False, 1e-4), (True, 0.03)):
        for a, b in zip(run(layer, "cuda", torch.float32, low), want):
            assert _off(a, b) < bound


@pytest.mark.gpu
def test_a_denoiser_whose_coordinates_have_a_gradient():
    torch.manual_seed(2)
    model = EDMModel(d_model=64, n_heads=2, n_layers=2, attn_types=["mha", "mha"], mlp_type="gated", rotary=RotaryPositions(12, axes=3, base=20.0))
    for p in model.parameters():
        if not p.any():
            torch.nn.init.normal_(p, std=0.1)
    g = torch.Generator().manual_seed(3)
    atoms, coords, sigma = torch.randn(2, 9, 6, generator=g), torch.randn(2, 9, 3, generator=g), torch.tensor([0.5, 1.5])
    pad = torch.arange(9)[None, :] >= torch.tensor([[9], [6]])

    def run(model, device, dtype):
        c = coords.to(device, dtype).requires_grad_()
        a, d = model(atoms.to(device, dtype), c, pad.to(device), sigma.to(device, dtype))
        assert d.isfinite().all()
        return torch.autograd.grad(a.square().sum(), c)[0]  # (the head's own gradient is not a number: an atom's distance to itself)

    want = run(model, "cpu", torch.float32)  # (the head forms distances in fp32 everywhere)
    assert _off(run(model.cuda(), "cuda", torch.float32), want) < 1e-4


@pytest.mark.gpu
def test_coordinates_of_16_bits_and_without_grad_mode():
    layer, (x, pos, pad, _) = _layer().cuda().bfloat16(), _inputs()
    x, pad = x.cuda().bfloat16(), pad.cuda()
    for mask in (pad, pad.flip(1)):
        for dtype in (torch.bfloat16, torch.float16):
            low = pos.cuda().to(dtype)
            with torch.no_grad():
                want = layer(x, key_padding_mask=mask, positions=low.float())
                got = layer(x, key_padding_mask=mask, positions=low)
                also = layer(x, key_padding_mask=mask, positions=low.float().requires_grad_())
            real = ~mask
            assert torch.equal(got[real], want[real]) and torch.equal(also[real], want[real])
    q = torch.randn(1, 2, 20, 24, device="cuda")
    with torch.no_grad():  # a gradient that nobody forms is none
        p = pos[0].cuda().requires_grad_()
        assert torch.equal(mfb.rotary_embedding(q, None, p, ROTARY.frequencies)[0], mfb.rotary_embedding(q, None, p.detach(), ROTARY.frequencies)[0])
    with pytest.raises(ValueError, match="no gradient"):
        mfb.rotary_embedding(q, None, p, ROTARY.frequencies)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), 1e30])
def test_positions_of_padded_tokens_reach_nobody(device, value):
    """The dense core masks scores, which a NaN among the keys would survive."""
    layer, (x, pos, pad, dy) = _layer().to(device), _inputs()
    x, pos, pad, dy = (t.to(device) for t in (x, pos, pad, dy))
    for mask, g in ((pad, dy), (pad.flip(1), dy.flip(1))):
        outs = []
        for p in (pos, pos.masked_fill(mask[..., None], value)):
            leaf = x.clone().requires_grad_()
            y = layer(leaf, key_padding_mask=mask, positions=p)
            outs.append([y.masked_fill(mask[..., None], 0.0), torch.autograd.grad(y, leaf, g)[0]])
        assert torch.equal(outs[0][0], outs[1][0])
        real = ~mask
        assert torch.equal(outs[0][1][real], outs[1][1][real]) and outs[1][1].isfinite().all()


def test_layers_of_an_earlier_version():
    """A module that was stored whole before there were rotary positions has no such attribute."""
    torch.manual_seed(4)
    trunk = TransformerTrunk(32, 4, ["mha"])
    x, cond = torch.randn(2, 5, 32), torch.randn(2, 32)
    want = trunk(x, cond)
    state = pickle.dumps(trunk)
    old = pickle.loads(state)
    for m in old.modules():
        m.__dict__.pop("rotary", None)
    assert torch.equal(old(x, cond), want)


def test_frequencies_first_asked_for_in_inference_mode():
    """They are made once and kept: as ordinary tensors, whoever asks first."""
    rotary = RotaryPositions(rotary_dim=12, axes=3)
    with torch.inference_mode():
        rotary.frequencies
    pos = torch.randn(1, 4, 3, requires_grad=True)
    y = rotate_torch(torch.randn(1, 2, 4, 16), pos, rotary.frequencies)
    assert torch.autograd.grad(y.sum(), pos)[0].isfinite().all()


def test_unknown_layouts_are_refused_on_the_cpu_too():
    x, pos, table = torch.ones(1, 1, 3, 8), torch.arange(3), mfb.rotary_frequencies(8)
    with pytest.raises(ValueError, match="layout must be one of"):
        rotate_torch(x, pos, table, "halves")
    with pytest.raises(ValueError, match="layout must be one of"):
        RotaryPositions(8, layout="Half")
    with pytest.raises(ValueError, match="amplitude must be finite"):
        RotaryPositions(8, amplitude=float("nan"))


def test_a_layer_takes_every_argument_of_the_frequencies():
    more = dict(axes=1, base=500.0, scaling="parts", factor=4.0, original_length=64.0, slow=0.5, fast=3.0)
    want = mfb.rotary_frequencies(32, **more)
    assert torch.equal(RotaryPositions(32, **more).frequencies, want)
    assert not torch.equal(mfb.rotary_frequencies(32, **{**more, "slow": 1.0, "fast": 32.0}), want)
