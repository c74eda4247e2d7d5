"""Captured training passes over leaves whose gradients another stream takes, as under a data-parallel wrapper."""
import pytest
import torch

import matterformer_b200 as mfb
from matterformer_b200.dp import GraphedTrainStep
from matterformer_b200.rotary import RotaryPositions
from matterformer_b200.synthetic import config5_batch
from matterformer_b200.trunk import EDMLoss, EDMModel, EDMPreconditioner

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _gradient_nodes(leaves, stream):
    """The nodes that take the leaves' gradients, made on `stream`; what holds them keeps them alive."""
    with torch.cuda.stream(stream):
        return [t.expand_as(t).grad_fn.next_functions[0][0] for t in leaves]


def _ops(wide):
    g = torch.Generator().manual_seed(0)
    x, *params = [(torch.randn(*s, generator=g) * 0.1).to(BF16).cuda() for s in ((40, 64), (144, 64), (64, 72), (144,), (64,))]
    return [t.requires_grad_() for t in (x, *(p.float() if wide else p for p in params))]


@pytest.mark.parametrize("wide", [False, True], ids=["bf16", "fp32 parameters"])
@pytest.mark.parametrize("how", ["backward", "grad"])
def test_the_block(how, wide):
    leaves = _ops(wide)
    pos, table = torch.arange(40).cuda(), mfb.rotary_frequencies(64)

    def step():
        y = mfb.gated_mlp(mfb.rotary_embedding(leaves[0].view(1, 1, 40, 64), None, pos, table)[0], *leaves[1:])
        loss = y.float().square().sum()
        if how == "grad":
            return torch.autograd.grad(loss, leaves)
        for t in leaves:
            t.grad = None
        loss.backward()
        return [t.grad for t in leaves]

    owner, capture = torch.cuda.Stream(), torch.cuda.Stream()
    held = _gradient_nodes(leaves, owner)
    capture.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(capture):
        for _ in range(2):
            want = [g.clone() for g in step()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=capture):
        got = step()
    for g in got:
        g.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert len(held) == 5 and all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_training_step():
    """The denoiser with gated blocks and rotary positions is captured, and every parameter gets a gradient."""
    torch.manual_seed(1)
    net = EDMPreconditioner(EDMModel(d_model=128, n_heads=2, n_layers=2, mlp_type="gated", rotary=RotaryPositions(48, axes=3, base=50.0))).cuda()
    for p in net.parameters():
        if not p.any():
            torch.nn.init.normal_(p, std=0.05)
    held = _gradient_nodes(list(net.parameters()), torch.cuda.Stream())
    opt = torch.optim.AdamW(net.parameters(), lr=0.0, fused=True, capturable=True)
    batch = {k: v.cuda() for k, v in config5_batch(8, seed=2).items() if k != "num_atoms"}
    step = GraphedTrainStep(net, EDMLoss(sigma_data=1.0), opt, batch, warmup=3, clip=0.0)
    step()
    torch.cuda.synchronize()
    assert held and torch.isfinite(step.loss) and all(p.grad.isfinite().all() and p.grad.any() for p in net.parameters())
