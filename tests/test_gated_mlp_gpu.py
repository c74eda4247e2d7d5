"""Gated feed-forward block against its definition in 64 bits."""
import pytest
import torch

import matterformer_b200 as mfb

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _operands(rows, C, F, O, dtype, bias, seed=0, lead=()):
    g = torch.Generator().manual_seed(seed)

    def r(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()

    ops = [r(*lead, rows, C), r(2 * F, C, scale=C**-0.5), r(O, F, scale=F**-0.5)]
    ops += [r(2 * F, scale=0.1), r(O, scale=0.1)] if bias else [None, None]
    return ops, r(*lead, rows, O)


def _exact(ops, dy, act):
    ops = [None if t is None else t.detach().double().requires_grad_() for t in ops]
    x, w_in, w_out, b_in, b_out = ops
    gate, up = torch.nn.functional.linear(x, w_in, b_in).chunk(2, dim=-1)
    f = torch.nn.functional.silu(gate) if act == "silu" else torch.nn.functional.gelu(gate, approximate="tanh")
    y = torch.nn.functional.linear(f * up, w_out, b_out)
    return [y.detach(), *torch.autograd.grad(y, [t for t in ops if t is not None], dy.double())]


def _off(got, want):
    """Root mean square of the difference over that of the result."""
    return ((got.double() - want).norm() / want.norm().clamp_min(1e-300)).item()


# Roundings on the way to a result, each at most u = eps / 2 of its value: forward the hidden value and the result, 2 u; backward the
# pre-activations (a factor 1 + z f''/f' <= 2.4 for the gate where the slope is not near its zero, and one for the up side), the gradient of the
# pre-activations, and the result.  Independent roundings add in squares, so 6 u bounds the root mean square with room for the zero
# of the slope; fp32 sums of up to some thousand products add less than a tenth of a bf16 u.
def _bound(dtype):
    return 6 * torch.finfo(dtype).eps / 2


def _run(ops, dy, act):
    leaves = [None if t is None else t.detach().requires_grad_() for t in ops]
    y = mfb.gated_mlp(*leaves, activation=act)
    return [y.detach(), *torch.autograd.grad(y, [t for t in leaves if t is not None], dy)]


SIZES = [(1, 8, 8, 8), (7, 64, 128, 64), (29, 512, 2048, 512), (128, 72, 136, 200), (129, 512, 1368, 512), (257, 200, 72, 328), (300, 1024, 264, 512),
         (1000, 520, 1032, 264), (4096, 64, 256, 64), (9, 4096, 80, 2048)]  # fmt: skip


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("rows,C,F,O", SIZES)
def test_forward_and_gradients(rows, C, F, O, dtype):
    act, bias = ("silu", "gelu_tanh")[(rows + C) % 2], (rows + F // 8) % 3 != 0
    ops, dy = _operands(rows, C, F, O, dtype, bias)
    got, want = _run(ops, dy, act), _exact(ops, dy, act)
    assert mfb.gated_mlp_status() == 0
    for i, (a, b) in enumerate(zip(got, want)):
        assert a.shape == b.shape and a.dtype == dtype
        assert _off(a, b) < _bound(dtype), f"output {i}: {_off(a, b):.2e}"
    with torch.no_grad():  # nothing kept for a backward pass
        assert torch.equal(mfb.gated_mlp(*ops, activation=act), got[0])
