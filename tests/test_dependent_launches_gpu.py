"""Every kernel that may begin before the one ahead of it has ended, straight behind one that lets it, back to back in a graph.

The rotation of a tensor announces its successor when it begins; what it makes is the operand of the kernel under test, at the same place in
memory round after round, so that a value read too soon is the last round's.
"""
import pytest
import torch

import matterformer_b200 as mfb
from matterformer_b200 import fused
from matterformer_b200.sparse import build_radius_blocks, local_window_attention_packed

pytestmark = pytest.mark.gpu

ROUNDS = 10


def _turn(t):
    """Another tensor of the same shape, by the rotary kernel alone."""
    pairs = t.shape[-1] // 2
    flat = t.reshape(1, 1, -1, t.shape[-1])
    places = _turn.places.setdefault(flat.shape[2], torch.arange(flat.shape[2], dtype=torch.int32, device=t.device) % 7)
    return mfb.rotary_embedding(flat, None, places, torch.full((min(pairs, 128),), 0.3, dtype=torch.float64))[0].view(t.shape)


_turn.places = {}


def _case(name):
    """(shape, type) of the operand, and what is made of it: tensors."""
    g = torch.Generator().manual_seed(0)

    def r(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()

    BF, B, N, C = torch.bfloat16, 256, 29, 512
    x, gate, shift = r(B, N, C, dtype=BF), r(B, C), r(B, C)
    pad = (torch.arange(N)[None, :] >= torch.randint(5, N + 1, (B, 1), generator=g)).cuda()
    valid = ~pad
    ones = torch.ones_like(valid)
    b, n = 16, 100
    large = torch.ones(b, n, dtype=torch.bool).cuda()
    heads, tall = [r(B, 4, N, 64, dtype=BF, scale=0.3) for _ in range(5)], [r(b, 4, n, 64, dtype=BF, scale=0.3) for _ in range(5)]
    bias = [r(B, 4, N, N), r(B, 4, N, N), r(B, 4, N, N), r(B, 4, N)]
    residual = [r(B, 4, N, N, 16, scale=0.2), r(B, 4, N, N, 16, scale=0.2), r(B, 4, N)]
    tall_bias, atoms = (r(b, 4, n, n), r(b, 4, n, n), r(b, 4, n, n), r(b, 4, n)), r(B, N, 3)
    counts, long, cells = valid.sum(1).int(), torch.full((8,), 1000, dtype=torch.int32).cuda(), torch.full((8,), 400, dtype=torch.int32).cuda()
    lattice = torch.tensor([[1.3, 1.4, 1.5, 0.1, -0.05, 0.2]]).repeat(8, 1).cuda()
    w_rbf, w_out, b_out, centers = r(128, 16), r(128), r(1), torch.linspace(0, 4, 16).cuda()
    noise, weight, wide_bias = r(B), r(512, 7), r(512)

    def simplicial(ops, valid, **more):
        return mfb.simplicial_attention_cuda(*ops, query_valid=valid, pair_key_valid=valid, **more)

    def simplicial_back(ops, valid, **more):
        """Past autograd, whose stream of the forward pass would be another than the capture's."""
        named = dict(zip(("u", "v_bias", "w", "gate"), more.get("factorized_bias", ())))
        named.update(zip(("angle_left", "angle_right", "angle_gate"), more.get("angle_residual", ())))
        _, lse, out = mfb.cuda_simplicial_attention_forward(*ops, query_valid=valid, pair_key_valid=valid, pair_valid=None, **named)
        wanted = {k: True for k in ("need_du", "need_dv_bias", "need_dw", "need_dgate") if "u" in named}
        return lambda dy: [t for t in mfb.cuda_simplicial_attention_backward(dy, *ops, out, lse, query_valid=valid, pair_key_valid=valid, pair_valid=None,
                                                                             **named, **wanted) if t is not None]  # fmt: skip

    def function_back(function, saved, *args):
        """The backward pass of one of the framework's autograd functions on a context of its own."""

        class Context:
            needs_input_grad = (True,) * len(args)

            def save_for_backward(self, *t):
                self.saved_tensors = t

            def mark_non_differentiable(self, *_):
                pass

        ctx = Context()
        function.forward(ctx, *args)
        return lambda dy: [t for t in function.backward(ctx, *([dy] * saved)) if t is not None]

    cases = {
        "gated_residual": ((B, N, C), BF, lambda t: fused.gated_residual(x, gate, t, pad)),
        "gated_residual of the stream": ((B, N, C), BF, lambda t: fused.gated_residual(t, gate, x)),
        "gated_residual backward": ((B, N, C), BF, function_back(fused._GatedResidual, 1, x, gate, x, pad)),
        "ln_modulate": ((B, N, C), BF, lambda t: fused.ln_modulate(t, shift, gate, eps=1e-6, out_dtype=BF)),
        "ln_modulate backward": ((B, N, C), BF, function_back(fused._LnModulate, 1, x, shift, gate, 1e-6, BF)),
        "gated_ln_modulate": ((B, N, C), BF, lambda t: fused.gated_ln_modulate(x, gate, t, pad, shift, gate, eps=1e-6, out_dtype=BF)),
        "affine norm": ((B, N, C), BF, lambda t: fused.affine_layer_norm(t, shift[0], gate[0], 1e-6, BF)),
        "column_sums": ((B * N, C), BF, fused.column_sums),
        "column_sums in fp32": ((B * N, 256), torch.float32, fused.column_sums),
        "gelu": ((B * N, C), BF, fused.gelu_tanh_forward),
        "gelu backward": ((B * N, C), BF, lambda t: fused.gelu_tanh_backward(x.view(-1, C), t)),
        "band, molecules": ((B, N, 3 * 256), BF, lambda t: local_window_attention_packed(t, 4, counts, window=64)),
        "band, wide tiles": ((8, 1000, 3 * 256), BF, lambda t: local_window_attention_packed(t, 4, long, window=64)),
        "small simplicial": ((B, 4, N, 64), BF, lambda t: simplicial([t, *heads[1:]], valid)),
        "small simplicial, keys": ((B, 4, N, 64), BF, lambda t: simplicial([heads[0], heads[1], heads[2], t, heads[4]], ones)),
        "small simplicial, residual": ((B, 4, N, N, 16), torch.float32, lambda t: simplicial(heads, valid, angle_residual=(t, *residual[1:]))),
        "small simplicial, bias": ((B, 4, N, N), torch.float32, lambda t: simplicial(heads, valid, factorized_bias=(t, *bias[1:]))),
        "small simplicial backward": ((B, 4, N, 64), BF, simplicial_back(heads, valid)),
        "small simplicial backward, residual": ((B, 4, N, 64), BF, simplicial_back(heads, valid, angle_residual=residual)),
        "rows backward": ((b, 4, n, 64), BF, simplicial_back(tall, large)),
        "trilinear": ((b, 4, n, 64), BF, lambda t: simplicial([t, *tall[1:]], large, factorized_bias=tall_bias)),
        "trilinear backward": ((b, 4, n, 64), BF, simplicial_back(tall, large, factorized_bias=tall_bias)),
        "block list": ((8, 400, 3), torch.float32, lambda t: (lambda made: [made.perm, made.block_count, made.block_cols, made.block_mask])(build_radius_blocks(t, lattice, cells, 2.0))),
        "token projection": ((B, N, 6), torch.float32, lambda t: fused.token_projection(t, noise, pad, weight, wide_bias)),
        "token projection backward": ((B, N, C), BF, function_back(fused._TokenProjection, 1, r(B, N, 6), noise, pad, weight, wide_bias)),
        "masked sum": ((B, N, 3), torch.float32, lambda t: fused.masked_update(pad, t, 2.0, center=True)),
        "pair head": ((B, N, 128), torch.float32, lambda t: fused.equivariant_pair_head(t, t, atoms, valid, w_rbf, w_out, b_out, centers, 1.0)),
        "noise levels": ((1024, 2), torch.float32, lambda t: [*fused.edm_scalings(t.view(-1), 1.0), fused.noise_channel(t.view(-1))]),
        "time embedding": ((512, 2), torch.float32, lambda t: fused.time_embedding(t.view(-1), 256, BF)),
    }
    return cases[name]


NAMES = ["affine norm", "band, molecules", "band, wide tiles", "block list", "column_sums", "column_sums in fp32", "gated_ln_modulate", "gated_residual",
         "gated_residual backward", "gated_residual of the stream", "gelu", "gelu backward", "ln_modulate", "ln_modulate backward", "masked sum", "noise levels",
         "pair head", "rows backward", "small simplicial", "small simplicial backward", "small simplicial backward, residual", "small simplicial, bias",
         "small simplicial, keys", "small simplicial, residual", "time embedding", "token projection", "token projection backward", "trilinear",
         "trilinear backward"]  # fmt: skip


def _as_list(made):
    return [t for t in (made if isinstance(made, (list, tuple)) else [made]) if isinstance(t, torch.Tensor)]


@pytest.mark.parametrize("name", NAMES)
def test_straight_behind_a_rotation(name):
    shape, dtype, consume = _case(name)
    g = torch.Generator().manual_seed(1)
    inputs = [(torch.randn(*shape, generator=g) * 0.5).to(dtype).cuda() for _ in range(ROUNDS)]
    want = []
    for t in inputs:
        operand = _turn(t)
        torch.cuda.synchronize()
        want.append([w.clone() for w in _as_list(consume(operand))])
        torch.cuda.synchronize()
    assert all(w.float().isfinite().all() for made in want for w in made)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph, got = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(graph, stream=stream):
        for t in inputs:
            operand = _turn(t)
            got.append([w.clone() for w in _as_list(consume(operand))])
            del operand
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for x, y in zip(a, b, strict=True):
                assert torch.equal(x, y)


def test_behind_the_gated_block():
    """A gated residual and a column sum of the block's result, and the norm's backward pass of its input's gradient (frozen parameters)."""
    BF, g = torch.bfloat16, torch.Generator().manual_seed(2)

    def r(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g) * scale).to(BF).cuda()

    B, N, C, F = 64, 29, 512, 1368
    w_in, w_out, x, gate, shift = r(2 * F, C, scale=C**-0.5), r(C, F, scale=F**-0.5), r(B, N, C), r(B, C).float(), r(B, C).float()
    inputs = [r(B, N, C) for _ in range(ROUNDS)]

    def forward(t):
        y = mfb.gated_mlp(t, w_in, w_out)
        torch.cuda.synchronize() if forward.slow else None
        return [fused.gated_residual(x, gate, y), fused.column_sums(mfb.gated_mlp(t, w_in, w_out).view(-1, C))]

    def backward(t):
        leaf = t.detach().requires_grad_()
        y = mfb.gated_mlp(fused.ln_modulate(leaf, shift, gate, eps=1e-6, out_dtype=BF), w_in, w_out)
        return list(torch.autograd.grad(y, leaf, x))

    forward.slow = True
    want = [[w.clone() for w in forward(t) + backward(t)] for t in inputs]
    torch.cuda.synchronize()
    forward.slow = False
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph, got = torch.cuda.CUDAGraph(), []
    with torch.cuda.graph(graph, stream=stream):
        for t in inputs:
            got.append([w.clone() for w in forward(t) + backward(t)])
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            for u, v in zip(a, b, strict=True):
                assert torch.equal(u, v)
