"""A trunk with rotary positions and gated feed-forward blocks: the two operators together, as models call them."""
import pytest
import torch

from matterformer_b200.rotary import RotaryPositions
from matterformer_b200.sampler import edm_sample
from matterformer_b200.trunk import EDMLoss, EDMModel, EDMPreconditioner, GatedMlp, RegularAttention, TransformerTrunk, plan_sparse_attention

pytestmark = pytest.mark.gpu


def _trunk(layers, layout="half"):
    torch.manual_seed(0)
    trunk = TransformerTrunk(128, 4, layers, mlp_type="gated", rotary=RotaryPositions(rotary_dim=24, axes=3, base=50.0, layout=layout))
    for p in trunk.parameters():
        if not p.any():
            torch.nn.init.normal_(p, std=0.05)
    return trunk


def _inputs(B, N, seed=0):
    g = torch.Generator().manual_seed(seed)
    pad = torch.arange(N)[None, :] >= torch.randint(N // 2, N + 1, (B, 1), generator=g)
    return torch.randn(B, N, 128, generator=g), torch.randn(B, 128, generator=g), pad, torch.randn(B, N, 3, generator=g) * 2, torch.randn(B, N, 128, generator=g)


def _pass(trunk, device, inputs, dtype=None, **more):
    x, cond, pad, pos, dy = (t.to(device) for t in inputs)
    x.requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=dtype == "bf16"):
        y = trunk(x, cond, pad_mask=pad, positions=pos, **more)
    return [y.detach(), *torch.autograd.grad(y, [x, *trunk.parameters()], dy.to(y.dtype))]


def _off(a, b):
    return ((a.double().cpu() - b.double().cpu()).norm() / b.double().norm().clamp_min(1e-12).cpu()).item()


# Two layers of bf16 arithmetic against 64 bits: some ten roundings of 2^-9 in each (norm, projections, scores, probabilities, hidden values), each
# passed on with a factor near one, add in squares to 2^-9 * sqrt(20) = 0.9 %; gradients see them twice: 3 %.
@pytest.mark.parametrize("B,N", [(6, 29), (3, 70)])  # the small-molecule core, and the dense one
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_against_64_bits(B, N, layout):
    trunk, inputs = _trunk(["mha", "mha"], layout), _inputs(B, N)
    want = _pass(trunk.double(), "cpu", [t.double() if t.is_floating_point() else t for t in inputs])
    got = _pass(trunk.float().cuda(), "cuda", inputs, "bf16")
    assert _off(got[0], want[0]) < 0.015
    for a, b in zip(got[1:], want[1:]):
        assert a.isfinite().all() and _off(a, b) < 0.03
    assert all(block.attn._last_core_used == ("cuda" if N <= 32 else "torch") for block in trunk.blocks)


def test_fp32_is_exact():
    """Without 16-bit arithmetic the block's plain form and the rotation in 32 bits."""
    trunk, inputs = _trunk(["mha", "mha"]), _inputs(4, 20)
    want = _pass(trunk.double(), "cpu", [t.double() if t.is_floating_point() else t for t in inputs])
    got = _pass(trunk.float().cuda(), "cuda", inputs)
    for a, b in zip(got, want):
        assert _off(a, b) < 1e-4


@pytest.mark.parametrize("kind", ["radius", "local"])
def test_crystal_plans(kind):
    """Rotary positions before the sparse cores; shifting all of them changes nothing."""
    trunk = _trunk(["mha"]).cuda()
    x, cond, pad, pos, _ = (t.cuda() for t in _inputs(2, 100, seed=1))
    frac = torch.rand(2, 100, 3, generator=torch.Generator().manual_seed(2)).cuda()
    lattice = torch.tensor([[2.3, 2.4, 2.5, 0.1, -0.05, 0.2]]).repeat(2, 1).cuda()
    plan = plan_sparse_attention(frac, lattice, pad, 4.0, kind=kind)
    with torch.no_grad():
        a = trunk(x, cond, pad_mask=pad, sparse_plan=plan, positions=pos)
        b = trunk(x, cond, pad_mask=pad, sparse_plan=plan, positions=pos + 1.5)
        c = trunk(x, cond, pad_mask=pad, sparse_plan=plan, positions=2 * pos)
    assert trunk.blocks[0].attn._last_core_used == kind
    assert _off(b, a) < 1e-4 and _off(c, a) > 1e-3


def test_denoiser_step_and_sampling():
    """A training step with gradients for every parameter, and a captured sampling run."""
    torch.manual_seed(3)
    model = EDMModel(d_model=128, n_heads=2, n_layers=2, mlp_type="gated", rotary=RotaryPositions(rotary_dim=48, axes=3, base=50.0))
    net = EDMPreconditioner(model, sigma_data=1.0).cuda()
    for p in net.parameters():
        if not p.any():
            torch.nn.init.normal_(p, std=0.05)
    B, N = 5, 17
    pad = torch.arange(N)[None, :] >= torch.tensor([17, 9, 12, 3, 1])[:, None]
    types, coords = torch.randint(0, 5, (B, N)), torch.randn(B, N, 3)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss, _ = EDMLoss(sigma_data=1.0)(net, types.cuda(), coords.cuda(), pad.cuda())
    grads = torch.autograd.grad(loss, list(net.parameters()))
    assert loss.isfinite() and all(g.isfinite().all() for g in grads) and all(g.any() for g in grads)
    net.eval()
    torch.manual_seed(4)
    eager = edm_sample(net, torch.tensor([17, 9, 3]), num_steps=3, autocast_dtype=torch.bfloat16, use_cuda_graph=False)
    torch.manual_seed(4)
    captured = edm_sample(net, torch.tensor([17, 9, 3]), num_steps=3, autocast_dtype=torch.bfloat16, use_cuda_graph=True)
    assert torch.equal(eager[0], captured[0]) and torch.equal(eager[1], captured[1])


def test_gated_module_paths():
    """Widths that the kernels do not take, a 16-bit module, and fp32 parameters under autocast: one function."""
    torch.manual_seed(5)
    x = torch.randn(3, 40, 64)
    for hidden in (72, 70):
        module = GatedMlp(64, hidden=hidden, activation="gelu_tanh")
        want = module.double()(x.double())
        module = module.float().cuda()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            assert _off(module(x.cuda()), want) < 0.015
        assert _off(module(x.cuda()), want) < 1e-5
        assert _off(module.bfloat16()(x.cuda().bfloat16()), want) < 0.015


def test_attention_layer_without_positions_is_unchanged():
    layer = RegularAttention(128, 4).cuda()
    x = torch.randn(2, 20, 128, device="cuda")
    pad = torch.zeros(2, 20, dtype=torch.bool, device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = layer(x, key_padding_mask=pad)
    assert layer._last_core_used == "cuda" and y.shape == x.shape
