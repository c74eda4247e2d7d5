"""Rotary positions against their definition in 64 bits."""
import math

import pytest
import torch

import matterformer_b200 as mfb

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _exact(x, positions, table, layout, amplitude=1.0):
    """x (B, H, N, D) in 64 bits, pair by pair."""
    B, H, N, D = x.shape
    x = x.double()
    table = table.double().reshape(-1, table.shape[-1])
    pos = positions.double().cpu().reshape(-1, N, table.shape[0])
    angle = (pos[..., None] * table).reshape(-1, 1, N, table.numel()).to(x.device)
    cos, sin = amplitude * torch.cos(angle), amplitude * torch.sin(angle)
    P = table.numel()
    first = torch.arange(P) if layout == "half" else 2 * torch.arange(P)
    second = first + (P if layout == "half" else 1)
    out = x.clone()
    out[..., first] = x[..., first] * cos - x[..., second] * sin
    out[..., second] = x[..., first] * sin + x[..., second] * cos
    return out


def _close(got, want, size):
    """One rounding of the result, half a step of its value, and the error of sine and cosine in 32 bits (two units in the last place
    each, and half a unit of an angle of up to pi that is rounded to 32 bits) times the pair's length, at most ``size``."""
    u = torch.finfo(got.dtype).eps / 2
    err = (got.double() - want).abs()
    allowed = u * 1.001 * want.abs() + size * (2 * 2.0**-23 + math.pi * 2.0**-24 + 2 * 2.0**-24) * 1.5 + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    assert (err <= allowed).all(), f"off by {(err - allowed).max().item():.2e} more than allowed"


def _randn(g, *shape, dtype):
    return torch.randn(*shape, generator=g).to(dtype).cuda()


CASES = [  # B, H, K, N, D, rotary_dim, axes, layout
    (1, 1, 1, 1, 2, 2, 1, "half"), (1, 1, 1, 1, 2, 2, 1, "interleaved"), (2, 3, 1, 5, 10, 6, 1, "half"), (2, 3, 1, 5, 10, 6, 1, "interleaved"),
    (3, 8, 8, 29, 64, 48, 3, "half"), (3, 8, 2, 29, 64, 48, 3, "interleaved"), (2, 4, 4, 33, 64, 64, 1, "half"), (64, 8, 2, 1, 128, 128, 1, "half"),
    (1, 2, 2, 700, 80, 36, 3, "interleaved"), (1, 4, 1, 257, 40, 20, 1, "half"), (2, 2, 2, 40, 256, 256, 1, "interleaved"), (1, 1, 1, 3, 600, 2, 1, "half"),
]  # fmt: skip


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("B,H,K,N,D,rotary_dim,axes,layout", CASES)
def test_heads(B, H, K, N, D, rotary_dim, axes, layout, dtype):
    g = torch.Generator().manual_seed(B + H + N + D)
    table = mfb.rotary_frequencies(rotary_dim, axes=axes, base=100.0 if axes > 1 else 10000.0)
    pos = (torch.randn(B, N, axes, generator=g) * 3).cuda() if axes > 1 else torch.arange(N).cuda() + 11
    q, k = (_randn(g, B, h, N, D, dtype=dtype).requires_grad_() for h in (H, K))
    gq, gk = _randn(g, B, H, N, D, dtype=dtype), _randn(g, B, K, N, D, dtype=dtype)
    out = mfb.rotary_embedding(q, k, pos, table, layout=layout, amplitude=1.25)
    grads = torch.autograd.grad(out, (q, k), (gq, gk))
    for x, y, dy, dx in zip((q, k), out, (gq, gk), grads):
        assert y.shape == x.shape and y.dtype == dtype
        _close(y.detach(), _exact(x.detach(), pos, table, layout, 1.25), 1.25 * 1.5 * x.detach().abs().max().item())
        # the transposed rotation: the gradient of sum(dy * rotate(x))
        ref = x.detach().double().requires_grad_()
        want = torch.autograd.grad(_exact(ref, pos, table, layout, 1.25), ref, dy.double())[0]
        _close(dx, want, 1.25 * 1.5 * dy.abs().max().item())
