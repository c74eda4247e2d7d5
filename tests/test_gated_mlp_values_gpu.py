"""Gated feed-forward block: values that a kept pre-activation has to survive, and how close its results are."""
import pytest
import torch
import torch.nn.functional as F

import matterformer_b200 as mfb

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def _operands(rows, C, H, O, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    shapes = ((rows, C), (2 * H, C), (O, H), (2 * H,), (O,), (rows, O))
    scales = (1.0, C**-0.5, H**-0.5, 0.1, 0.1, 1.0)
    *ops, dy = [(torch.randn(*s, generator=g) * f).to(dtype).cuda() for s, f in zip(shapes, scales)]
    return ops, dy


def _run(ops, dy, act="silu"):
    leaves = [t.detach().requires_grad_() for t in ops]
    y = mfb.gated_mlp(*leaves, activation=act)
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)]


def _exact(ops, dy, act="silu"):
    ops = [t.detach().double().requires_grad_() for t in ops]
    gate, up = F.linear(ops[0], ops[1], ops[3]).chunk(2, dim=-1)
    y = F.linear((F.silu(gate) if act == "silu" else F.gelu(gate, approximate="tanh")) * up, ops[2], ops[4])
    return [y.detach(), *torch.autograd.grad(y, ops, dy.double())]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("rows", [16, 300])
def test_a_nan_token_has_nan_gradients(rows, dtype):
    """All pre-activations of a token are NaN: so is its gradient, and nobody else's."""
    ops, dy = _operands(rows, 64, 72, 80, dtype, 1)
    clean = _run(ops, dy)
    ops[0][3] = float("nan")
    y, dx, dw_in, dw_out, db_in, db_out = _run(ops, dy)
    keep = torch.arange(rows) != 3
    assert y[3].isnan().all() and dx[3].isnan().all()
    assert torch.equal(y[keep], clean[0][keep]) and torch.equal(dx[keep], clean[1][keep])
    assert dw_in.isnan().all() and dw_out.isnan().all() and db_in.isnan().all() and torch.equal(db_out, clean[5])


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("rows", [16, 300])
@pytest.mark.parametrize("side", ["gate", "up"])
def test_a_nan_bias_reaches_its_gradient(rows, side, dtype):
    """One channel's pre-activation is NaN in every token.  Of the gate it reaches both gradients of the channel, of the up side the gate's; the
    other groups of 16 channels of the token's kept values are untouched (in bf16 the other channels of its own as well)."""
    ops, dy = _operands(rows, 64, 80, 72, dtype, 2)
    clean = _run(ops, dy)[4]
    at = 21
    ops[3][at if side == "gate" else 80 + at] = float("nan")
    got = _run(ops, dy)[4]
    assert got[at].isnan()
    assert got[80 + at].isnan() if side == "gate" else got[80 + at] == clean[80 + at]
    group = torch.arange(160) % 80 // 16 == at // 16 if dtype == F16 else torch.arange(160) % 80 == at
    assert torch.equal(got[~group], clean[~group])


@pytest.mark.parametrize("rows", [16, 300])
@pytest.mark.parametrize("outlier", [10, 13, 16])
def test_fp16_channels_beside_an_outlier(rows, outlier):
    """One channel's up projection is 2^outlier times its neighbours'.  In such a group the fp16 form keeps 12 bits, one more than fp16 has, down to 2^-13 of
    the power of two in the largest, and steps of 2^-24 of that below: a value of the others is off by 2^-12 of itself or half such a step.

    The gradient of the gate's rows is a sum over the tokens of dh act'(g) u x: of the error of u by steps, each token's at most, added in squares
    (twice for the room of a sum of few); of the roundings of its own, 6 of 2^-11 as for every gradient of the block; of the steps of 2^-24
    that fp16 itself ends at, in every token's gradient of the pre-activations and in the result."""
    ops, dy = _operands(rows, 64, 80, 72, F16, 3)
    ops[1] *= 0.25
    ops[1][80 + 5] *= 2.0**6  # the projection holds 2^6 of it, the neighbours are made smaller by the rest
    others = [c for c in range(16) if c != 5]
    ops[1][[80 + c for c in others]] *= 2.0 ** (6 - outlier)
    ops[3].zero_()
    ops[2][:, 5] *= 2.0**-6
    got, want = _run(ops, dy)[2], _exact(ops, dy)[2]
    gate, up = F.linear(ops[0].double(), ops[1].double()).chunk(2, dim=-1)
    s = torch.sigmoid(gate)
    slope = s * (1 + gate * (1 - s))
    dh = dy.double() @ ops[2].double()
    step = up[:, :16].abs().amax(dim=1, keepdim=True) * 2.0**-25
    of_steps = 2 * ((dh * slope)[:, :16] * step).square().t() @ ops[0].double().square()
    for c in others:
        off = (got[c].double() - want[c]).norm()
        assert off <= 6 * 2.0**-11 * want[c].norm() + of_steps[c].sum().sqrt() + 2.0**-24 * (rows * want.shape[1]) ** 0.5


@pytest.mark.parametrize("rows,C,H,O", [(29, 512, 2048, 512), (1000, 512, 1368, 512), (3000, 264, 1032, 520)])
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_distance_to_the_rounding_of_the_result_alone(rows, C, H, O, act, dtype):
    """Root mean square errors in units of what rounding the exact result gives.  Forward the hidden value and the result are rounded, independently:
    sqrt(2).  Backward the gradient of the pre-activations and the result are, and the kept pre-activations by 2^-k of a rounding, k = 3 in bf16,
    in fp16 2 and, in the 15 % of groups that have a value below 2^-7 of the power of two in their largest, 1.  For gates of unit variance f(z)
    takes that up 1.21 times (root mean square of z f'(z) over that of f), f'(z) 0.35 times, a product with the up side once more: at most
    sqrt(2 + 1.21^2 / 4^k) = 1.42 and 1.46.  6 % are for sums of a few hundred values.  Pre-activations in the block's own type, k = 0,
    would be at 1.86."""
    ops, dy = _operands(rows, C, H, O, dtype, 4)
    got, want = _run(ops, dy, act), _exact(ops, dy, act)
    for i, (a, b) in enumerate(zip(got, want)):
        alone = (b.to(dtype).double() - b).norm()
        assert (a.double() - b).norm() < (1.5 if dtype == BF16 else 1.55) * alone, f"output {i}: {((a.double() - b).norm() / alone).item():.2f}"


@pytest.mark.parametrize("rows", [2, 8, 16, 17, 32, 33, 257, 600])
def test_a_row_does_not_depend_on_later_rows(rows):
    """Other values behind a token change no bit of its result and of its gradient."""
    ops, dy = _operands(rows, 128, 264, 136, BF16, 5)
    first = _run(ops, dy)
    k = max(1, rows // 2)
    ops[0][k:] = 3 * ops[0][k:].flip(0) + 1
    dy[k:] = -2 * dy[k:].flip(0)
    second = _run(ops, dy)
    for i in (0, 1):
        assert torch.equal(first[i][:k], second[i][:k]) and not torch.equal(first[i][k:], second[i][k:])
