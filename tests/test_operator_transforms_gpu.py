"""The gated block and rotary positions under tracing, torch.func and forward-mode differentiation: what these see, they see in plain operations."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad
import torch.nn.functional as F
from torch.fx.experimental.proxy_tensor import make_fx

import matterformer_b200 as mfb
from matterformer_b200.rotary import rotate_torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _r(*shape, seed=0, scale=1.0, dtype=BF16):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


W_IN, W_OUT = (lambda: _r(144, 64, seed=1, scale=0.125)), (lambda: _r(64, 72, seed=2, scale=0.118))


def _block(x, w_in, w_out):
    gate, up = F.linear(x, w_in).chunk(2, dim=-1)
    return F.linear(F.silu(gate) * up, w_out)


def _off(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


# In plain bf16 operations each of gate, up, activation, product and result is rounded, at most 2^-8 each: five in squares, and with the
# tangent's or gradient's own five and the products of a derivative at most twenty: 2^-8 sqrt(20).
BOUND = 2.0**-8 * 20**0.5


def _traced(how, f, x):
    return torch.jit.trace(f, (x,), check_trace=False) if how == "jit" else make_fx(f)(x)


@pytest.mark.parametrize("how", ["jit", "fx"])
@pytest.mark.parametrize("wide", [False, True], ids=["bf16", "fp32 parameters"])
def test_a_trace_of_the_block_follows_its_input(how, wide):
    w_in, w_out = (w.float() if wide else w for w in (W_IN(), W_OUT()))
    with torch.no_grad():
        f = _traced(how, lambda t: t + mfb.gated_mlp(t, w_in, w_out), _r(40, 64, seed=3))
        for rows_seed in (4, 5):
            x = _r(40, 64, seed=rows_seed)
            want = x.double() + _block(x.double(), w_in.double(), w_out.double())
            assert _off(f(x), want) < BOUND


@pytest.mark.parametrize("how", ["jit", "fx"])
def test_a_trace_keeps_the_type_under_autocast(how):
    """An fp16 block under bf16 autocast is one of fp16, traced or not."""
    w_in, w_out, x = W_IN().half(), W_OUT().half(), _r(40, 64, seed=12, dtype=torch.float16)
    with torch.no_grad(), torch.autocast("cuda", dtype=BF16):
        f = _traced(how, lambda t: mfb.gated_mlp(t, w_in, w_out), x)
        assert mfb.gated_mlp(x, w_in, w_out).dtype == torch.float16
    got = f(x)  # (a trace that runs under autocast is subject to it like any other operations)
    assert got.dtype == torch.float16
    assert _off(got, _block(x.double(), w_in.double(), w_out.double())) < BOUND / 8


def test_the_block_under_transforms():
    w_in, w_out = W_IN(), W_OUT()
    x, v = _r(3, 20, 64, seed=6), _r(3, 20, 64, seed=7)
    f = lambda t: mfb.gated_mlp(t, w_in, w_out)  # noqa: E731
    g = lambda t: _block(t, w_in.double(), w_out.double())  # noqa: E731
    assert _off(torch.func.vmap(f)(x), g(x.double())) < BOUND
    assert _off(torch.func.jvp(f, (x,), (v,))[1], torch.func.jvp(g, (x.double(),), (v.double(),))[1]) < BOUND
    assert _off(torch.func.grad(lambda t: (f(t).float() * v.float()).sum())(x), torch.func.grad(lambda t: (g(t) * v.double()).sum())(x.double())) < BOUND
    weights = torch.stack([w_in, -w_in])
    assert _off(torch.func.vmap(lambda w: mfb.gated_mlp(x[0], w, w_out))(weights)[1], _block(x[0].double(), -w_in.double(), w_out.double())) < BOUND
    with forward_ad.dual_level(), torch.no_grad():
        tangent = forward_ad.unpack_dual(f(forward_ad.make_dual(x, v))).tangent
    assert _off(tangent, torch.func.jvp(g, (x.double(),), (v.double(),))[1]) < BOUND


def _turns(packed):
    table, pos = mfb.rotary_frequencies(24, axes=3), _r(2, 9, 3, seed=8, dtype=torch.float32)
    if packed:
        return (2, 9, 3 * 2 * 32), lambda x: mfb.rotary_packed(x, 2, pos, table), pos
    return (2, 4, 9, 32), lambda x: mfb.rotary_embedding(x, x[:, :1], pos, table), pos


def _turned(packed, x, pos):
    table = mfb.rotary_frequencies(24, axes=3)
    if not packed:
        return torch.cat([rotate_torch(x, pos, table), rotate_torch(x[:, :1], pos, table)], dim=1)
    q, k, v = x.view(2, 9, 3, 2, 32).permute(2, 0, 3, 1, 4)
    return torch.stack([rotate_torch(q, pos, table), rotate_torch(k, pos, table), v]).permute(1, 3, 0, 2, 4).reshape(2, 9, -1)


def _whole(y):
    return y if isinstance(y, torch.Tensor) else torch.cat(list(y), dim=1)


# fp32: a product of two and a sum on either side, sines and cosines to a few units
TOL = dict(rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("packed", [False, True])
def test_rotary_under_traces_and_transforms(packed):
    shape, f, pos = _turns(packed)
    x, v = _r(*shape, seed=9, dtype=torch.float32), _r(*shape, seed=10, dtype=torch.float32)
    with torch.no_grad():
        for how in ("jit", "fx"):
            t = _traced(how, lambda x: _whole(f(x)) + 0, _r(*shape, seed=11, dtype=torch.float32))
            torch.testing.assert_close(t(x), _turned(packed, x, pos), **TOL)
    torch.testing.assert_close(torch.func.jvp(lambda x: _whole(f(x)), (x,), (v,))[1], _turned(packed, v, pos), **TOL)
    stacked = torch.stack([x, v])
    torch.testing.assert_close(torch.func.vmap(lambda x: _whole(f(x)))(stacked), torch.stack([_turned(packed, x, pos), _turned(packed, v, pos)]), **TOL)
    grad = torch.func.grad(lambda t: (_whole(f(t)).sin()).sum())(x)
    leaf = x.clone().requires_grad_()
    torch.testing.assert_close(grad, torch.autograd.grad(_turned(packed, leaf, pos).sin().sum(), leaf)[0], **TOL)
