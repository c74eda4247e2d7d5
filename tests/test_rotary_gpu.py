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


def _close(got, want, size, angle=0.0):
    """One rounding of the result, half a step of its value, and the error of sine and cosine in 32 bits (two units in the last place
    each, and half a unit of an angle of up to pi that is rounded to 32 bits) times the pair's length, at most ``size``.

    Angles of up to ``angle`` radians are products in 64 bits on both sides and no more exact than that: the oracle rounds
    position * frequency (2^-53 of the angle), the kernel frequency / 2 pi, its product with the position, and 2 pi itself (three times that).
    An angle's error moves a value by at most that times the pair's length.  At 2^40 and a frequency of 1 that is 5e-4."""
    u = torch.finfo(got.dtype).eps / 2
    err = (got.double() - want).abs()
    allowed = u * 1.001 * want.abs() + size * (2 * 2.0**-23 + math.pi * 2.0**-24 + 2 * 2.0**-24) * 1.5 + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    allowed = allowed + size * 4 * 2.0**-53 * angle
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


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("D,rotary_dim,layout", [(64, 2 * p, la) for p in (1, 2, 3, 4, 7, 8, 12, 16, 31, 32) for la in ("half", "interleaved")]
                         + [(72, 36, "half"), (20, 18, "half"), (20, 20, "interleaved"), (7, 4, "half"), (7, 6, "interleaved")])  # fmt: skip
def test_any_number_of_pairs(D, rotary_dim, layout, dtype):
    """Vectors of 16, 8, 4 bytes and single elements; pairs that begin or end inside a vector."""
    g = torch.Generator().manual_seed(D * rotary_dim)
    table = mfb.rotary_frequencies(rotary_dim)
    q, k = _randn(g, 2, 3, 37, D, dtype=dtype), _randn(g, 2, 2, 37, D, dtype=dtype)
    pos = torch.randint(0, 5000, (2, 37), generator=g, dtype=torch.int32).cuda()
    for x, y in zip((q, k), mfb.rotary_embedding(q, k, pos, table, layout=layout)):
        _close(y, _exact(x, pos, table, layout), 1.5 * x.abs().max().item())
        assert torch.equal(y[..., rotary_dim:], x[..., rotary_dim:])


@pytest.mark.parametrize("heads,D,rotary_dim,axes", [(8, 64, 48, 3), (3, 40, 22, 1), (1, 8, 8, 1), (5, 16, 12, 2)])
def test_packed_is_heads(heads, D, rotary_dim, axes):
    g = torch.Generator().manual_seed(heads)
    B, N = 5, 29
    table = mfb.rotary_frequencies(rotary_dim, axes=axes, base=50.0)
    pos = (torch.randn(B, N, axes, generator=g) if axes > 1 else torch.randn(B, N, generator=g)).cuda()
    qkv = _randn(g, B, N, 3 * heads * D, dtype=BF16).requires_grad_()
    dy = _randn(g, B, N, 3 * heads * D, dtype=BF16)
    y = mfb.rotary_packed(qkv, heads, pos, table)
    (dx,) = torch.autograd.grad(y, qkv, dy)
    q, k, v = qkv.detach().view(B, N, 3, heads, D).permute(2, 0, 3, 1, 4)
    tq, tk = mfb.rotary_embedding(q, k, pos, table)
    assert tq.stride(-1) == 1
    assert torch.equal(y.detach().view(B, N, 3, heads, D).permute(2, 0, 3, 1, 4), torch.stack([tq, tk, v]))
    gq, gk, gv = dy.view(B, N, 3, heads, D).permute(2, 0, 3, 1, 4)
    back = mfb.rotary_embedding(gq, gk, -pos, table)
    assert torch.equal(dx.view(B, N, 3, heads, D).permute(2, 0, 3, 1, 4), torch.stack([*back, gv]))


def test_strides_and_alignment():
    g = torch.Generator().manual_seed(1)
    table = mfb.rotary_frequencies(32)
    pos = torch.arange(50).cuda()
    x = _randn(g, 2, 4, 50, 40, dtype=BF16)
    want, _ = mfb.rotary_embedding(x, None, pos, table)
    token_major = x.transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.zeros(2, 4, 50, 61, dtype=BF16, device="cuda")
    wide[..., 3:43] = x
    every_other = torch.stack([x, x + 1], dim=-1)[..., 0]  # channels apart
    for other in (token_major, wide[..., 3:43], every_other, x.flip(2).flip(2)):
        y, none = mfb.rotary_embedding(other, None, pos, table)
        assert none is None and torch.equal(y, want)
    one_head = x[:, :1].expand(2, 4, 50, 40)  # a key head that queries share, as a view
    assert torch.equal(mfb.rotary_embedding(one_head, None, pos, table)[0], want[:, :1].expand(2, 4, 50, 40))
    y, _ = mfb.rotary_embedding(token_major, None, pos, table)
    assert y.stride() == token_major.stride()


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])
def test_far_positions(dtype):
    """Ten million places away, past 2^24, and negative: angles keep their digits."""
    g = torch.Generator().manual_seed(2)
    table = mfb.rotary_frequencies(64)
    x = _randn(g, 1, 2, 8, 64, dtype=dtype)
    for pos in (torch.tensor([10_000_019, 16_777_217, 2**31 + 11, 2**40 + 7, -5, 0, 1, -(2**33)]), torch.tensor([1e6 + 0.25, -3.5, 2.0**24, 7.75, 0.0, 1e-3, 12345.678, 99999.5])):
        y, _ = mfb.rotary_embedding(x, None, pos.cuda(), table)
        _close(y, _exact(x, pos, table, "half"), 1.5 * x.abs().max().item(), angle=pos.abs().max().item())


def test_position_types_and_sharing():
    g = torch.Generator().manual_seed(3)
    table, wide = mfb.rotary_frequencies(16), mfb.rotary_frequencies(18, axes=3)
    x = _randn(g, 4, 2, 11, 24, dtype=F32)
    pos = torch.randint(-100, 100, (4, 11), generator=g).cuda()
    want, _ = mfb.rotary_embedding(x, None, pos, table)
    for t in (torch.int32, torch.float32, torch.float64):
        assert torch.equal(mfb.rotary_embedding(x, None, pos.to(t), table)[0], want)
    assert torch.equal(mfb.rotary_embedding(x, None, pos[0], table)[0], mfb.rotary_embedding(x, None, pos[:1].repeat(4, 1), table)[0])
    three = torch.randn(11, 3, generator=g).cuda()
    assert torch.equal(mfb.rotary_embedding(x, None, three, wide)[0], mfb.rotary_embedding(x, None, three.repeat(4, 1, 1), wide)[0])
    strided = torch.stack([pos, pos], dim=-1)[..., 0]
    assert torch.equal(mfb.rotary_embedding(x, None, strided, table)[0], want)


def test_gradient_is_the_transpose_and_is_differentiable():
    """<dy, R x> = <R^T dy, x>; a rotation there and back; and the gradient's gradient."""
    g = torch.Generator().manual_seed(4)
    table = mfb.rotary_frequencies(24)
    q, dy, v = (_randn(g, 2, 3, 20, 32, dtype=F32) for _ in range(3))
    pos = torch.arange(20).cuda() * 7
    q.requires_grad_()
    dy.requires_grad_()
    y, _ = mfb.rotary_embedding(q, None, pos, table, amplitude=0.5)
    (dx,) = torch.autograd.grad(y, q, dy, create_graph=True)
    assert abs(((dy * y).sum() - (dx * q).sum()).item()) < 1e-5 * (dy.norm() * q.norm()).item()
    (ddy,) = torch.autograd.grad(dx, dy, v)
    assert torch.equal(ddy, mfb.rotary_embedding(v, None, pos, table, amplitude=0.5)[0])
    h = 0.5  # the operator is linear: a difference of any width
    difference = ((mfb.rotary_embedding(q + h * v, None, pos, table, amplitude=0.5)[0] - mfb.rotary_embedding(q - h * v, None, pos, table, amplitude=0.5)[0]) * dy).sum() / (2 * h)
    assert abs(difference.item() - (dx * v).sum().item()) < 1e-4 * (dy.norm() * v.norm()).item()


def test_one_of_two_outputs():
    g = torch.Generator().manual_seed(5)
    table, pos = mfb.rotary_frequencies(32), torch.arange(9).cuda()
    q, k = (_randn(g, 2, h, 9, 32, dtype=BF16).requires_grad_() for h in (4, 1))
    dy = _randn(g, 2, 1, 9, 32, dtype=BF16)
    _, tk = mfb.rotary_embedding(q, k, pos, table)
    dq, dk = torch.autograd.grad(tk, (q, k), dy, allow_unused=True)
    assert dq is None and torch.equal(dk, mfb.rotary_embedding(dy, None, -pos, table)[0])
    shared = dy[..., :1].expand(dy.shape)  # a broadcast gradient
    (dk,) = torch.autograd.grad(mfb.rotary_embedding(q, k, pos, table)[1], k, shared)
    assert torch.equal(dk, mfb.rotary_embedding(shared.contiguous(), None, -pos, table)[0])


def test_infinities_stay_in_their_pair():
    x = torch.ones(1, 1, 4, 16, dtype=F32, device="cuda")
    x[0, 0, 1, 2], x[0, 0, 2, 15], x[0, 0, 3, 9] = float("inf"), float("nan"), float("nan")
    for layout, partner in (("half", 8), ("interleaved", 3)):
        y, _ = mfb.rotary_embedding(x, None, torch.arange(4).cuda(), mfb.rotary_frequencies(12), layout=layout)
        bad = ~y.isfinite()
        P = 6
        want = torch.zeros_like(bad)
        want[0, 0, 1, 2] = want[0, 0, 1, 2 + P if layout == "half" else 3] = True
        want[0, 0, 2, 15] = True
        want[0, 0, 3, 9] = want[0, 0, 3, 9 - P if layout == "half" else 8] = True
        assert torch.equal(bad, want), layout


def test_empty():
    table = mfb.rotary_frequencies(8)
    for shape in ((0, 2, 3, 8), (2, 0, 3, 8), (2, 2, 0, 8)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        y, _ = mfb.rotary_embedding(x, None, torch.arange(shape[2]).cuda(), table)
        assert y.shape == x.shape and torch.autograd.grad(y.sum(), x)[0].shape == x.shape
    assert mfb.rotary_packed(torch.empty(0, 5, 48, device="cuda"), 2, torch.arange(5).cuda(), table).shape == (0, 5, 48)


def test_stream_and_capture():
    g = torch.Generator().manual_seed(6)
    table = mfb.rotary_frequencies(32)
    x, dy = _randn(g, 3, 2, 40, 32, dtype=BF16).requires_grad_(), _randn(g, 3, 2, 40, 32, dtype=BF16)
    pos = torch.arange(40).cuda()

    def call():
        y, _ = mfb.rotary_embedding(x, None, pos, table)
        return y.detach(), torch.autograd.grad(y, x, dy)[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    alive = mfb.rotary_embedding(x, None, pos, table)
    with pytest.raises(RuntimeError, match="release that graph"), torch.cuda.graph(torch.cuda.CUDAGraph()):
        call()
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    with torch.no_grad():
        x.mul_(2)
        pos.add_(100)
    graph.replay()
    for a, b in zip(out, call()):
        assert torch.equal(a, b)


def test_many_tokens_and_large_offsets():
    """More than 2^31 elements between the first and the last head."""
    N, D = 70_000, 64
    table = mfb.rotary_frequencies(64)
    base = torch.empty(2 * 520 * N * D, dtype=BF16, device="cuda")  # 9.3 GB
    x = base.view(1, 1040, N, D)[:, ::1039]  # the first and the last
    x.copy_(torch.randn(1, 2, N, D, device="cuda"))
    pos = torch.arange(N).cuda()
    y, _ = mfb.rotary_embedding(x, None, pos, table)
    assert torch.equal(y, mfb.rotary_embedding(x.contiguous(), None, pos, table)[0])


@pytest.mark.parametrize("inference", [False, True])
@pytest.mark.parametrize("how", ["native", "python"])
def test_positions_and_table_changed_before_the_backward_pass(how, inference, monkeypatch):
    """A changed table does not reach the gradient; changed positions are an error, or kept if nothing notes their changes."""
    if how == "python":
        monkeypatch.setattr(mfb._lib, "native", lambda: None)
    g = torch.Generator().manual_seed(9)
    with torch.inference_mode(inference):
        table, pos = mfb.rotary_frequencies(32), torch.arange(5).cuda()
    x, dy = _randn(g, 2, 3, 5, 32, dtype=F32).requires_grad_(), _randn(g, 2, 3, 5, 32, dtype=F32)
    want = torch.autograd.grad(mfb.rotary_embedding(x, None, pos, table)[0], x, dy)[0]
    y = mfb.rotary_embedding(x, None, pos, table)[0]
    with torch.inference_mode(inference):
        table.mul_(2)
    assert torch.equal(torch.autograd.grad(y, x, dy, retain_graph=True)[0], want)
    with torch.inference_mode(inference):
        pos.add_(1)
    if inference:
        assert torch.equal(torch.autograd.grad(y, x, dy)[0], want)
    else:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, x, dy)


@pytest.mark.parametrize("how", ["native", "python"])
def test_overlapping_windows(how, monkeypatch):
    """Tokens one element apart: their channels are adjacent, and no dense result has the same order of strides."""
    if how == "python":
        monkeypatch.setattr(mfb._lib, "native", lambda: None)
    g = torch.Generator().manual_seed(10)
    x = _randn(g, 2, 3, 75, dtype=F32).unfold(-1, 16, 1)
    table, pos = mfb.rotary_frequencies(16), torch.arange(60).cuda()
    y, z = mfb.rotary_embedding(x, x[:, :1].expand(2, 4, 60, 16), pos, table)
    _close(y, _exact(x, pos, table, "half"), 1.5 * x.abs().max().item())
    assert torch.equal(z, y[:, :1].expand(2, 4, 60, 16))


def test_sizes_beyond_the_kernel_are_refused():
    table, pos = mfb.rotary_frequencies(2), torch.zeros(1, device="cuda")
    x = torch.zeros(1, 1, 1, 2, device="cuda")
    for shape in ((2**31, 1, 1, 2), (2**32 + 1, 1, 1, 2), (1, 2**32 + 1, 1, 2), (1, 2**26 + 1, 1, 2)):
        with pytest.raises(ValueError, match="at most 2\\^27 elements a token"):
            mfb.rotary_embedding(x.expand(shape), None, pos, table)
        with pytest.raises(ValueError, match="at most 2\\^27 elements a token"):
            mfb.rotary_embedding(x, x.expand(shape), pos, table) if shape[0] == 1 else mfb.rotary_embedding(x.expand(shape), x.expand(shape), pos, table)
