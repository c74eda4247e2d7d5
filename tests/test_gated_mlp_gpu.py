"""Gated feed-forward block against its definition in 64 bits."""
import ctypes
import threading

import pytest
import torch

import matterformer_b200 as mfb
from matterformer_b200 import _lib, gated

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
         (1000, 520, 1032, 264), (4096, 64, 256, 64), (9, 4096, 80, 2048),
         (100, 64, 8200, 520), (30, 512, 8192, 72), (500, 72, 4104, 264)]  # (few tiles over many hidden channels: in slices)  # fmt: skip


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


def test_gradient_against_differences():
    """<gradient, direction> for every operand against a central difference of the loss in 64 bits."""
    ops, dy = _operands(40, 64, 96, 72, BF16, True, seed=3)
    grads = _run(ops, dy, "silu")[1:]
    g = torch.Generator().manual_seed(4)

    def loss(i, v, h):
        x, w_in, w_out, b_in, b_out = (t.double() + (h * v if j == i else 0) for j, t in enumerate(ops))
        gate, up = torch.nn.functional.linear(x, w_in, b_in).chunk(2, dim=-1)
        return (torch.nn.functional.linear(torch.nn.functional.silu(gate) * up, w_out, b_out) * dy.double()).sum().item()

    for i, t in enumerate(ops):
        v = torch.randn(t.shape, generator=g).double().cuda()
        difference = (loss(i, v, 1e-5) - loss(i, v, -1e-5)) / 2e-5
        # each entry of the gradient is off by at most _bound of the root mean square; the sum's errors add in squares, times the direction
        allowed = 6 * _bound(BF16) * grads[i].double().norm().item()
        assert abs((grads[i].double() * v).sum().item() - difference) < allowed + 1e-4 * abs(difference)


@pytest.mark.parametrize("wanted", [(0,), (1,), (2,), (3,), (4,), (0, 2), (1, 4), (1, 2, 3)])
def test_only_the_wanted_gradients(wanted):
    ops, dy = _operands(300, 64, 72, 80, BF16, True, seed=5)
    everything = _run(ops, dy, "silu")[1:]
    leaves = [t.detach().requires_grad_(i in wanted) for i, t in enumerate(ops)]
    y = mfb.gated_mlp(*leaves)
    got = torch.autograd.grad(y, [leaves[i] for i in wanted], dy)
    for i, g in zip(wanted, got):
        assert torch.equal(g, everything[i])


@pytest.mark.parametrize("rows", [5, 300])
def test_fp32_parameters(rows):
    """Their bf16 copies compute, their gradients are not rounded."""
    ops, dy = _operands(rows, 64, 136, 72, BF16, True, seed=6)
    wide = [ops[0], *(t.float() for t in ops[1:])]
    got, want = _run(wide, dy, "gelu_tanh"), _exact(ops, dy, "gelu_tanh")
    assert [t.dtype for t in got] == [BF16, BF16, F32, F32, F32, F32]
    low = _run(ops, dy, "gelu_tanh")
    for a, b, c in zip(got, want, low):
        assert _off(a, b) < _bound(BF16)
        assert torch.equal(a.to(BF16), c)  # the same sums, rounded


@pytest.mark.parametrize("rows", [1, 8, 9, 16, 17, 31, 32, 33, 255, 256, 257])
def test_token_counts(rows):
    """Around the sizes at which kernels and tiles change; a row's result does not depend on the rows after it."""
    ops, dy = _operands(rows, 128, 264, 136, BF16, True, seed=7)
    got, want = _run(ops, dy, "silu"), _exact(ops, dy, "silu")
    for a, b in zip(got, want):
        assert _off(a, b) < _bound(BF16)


def test_shapes_strides_and_alignment():
    ops, dy = _operands(12, 64, 72, 80, BF16, True, seed=8, lead=(2, 3))
    base = _run(ops, dy, "silu")
    assert base[0].shape == (2, 3, 12, 80) and base[1].shape == ops[0].shape
    x = ops[0]
    wide = torch.full((2, 3, 12, 130), float("nan"), dtype=BF16, device="cuda")
    wide[..., 3:67] = x
    shifted = [wide[..., 3:67], *(torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape) for t in ops[1:])]
    order = x.transpose(0, 2).contiguous().transpose(0, 2)
    for other in (shifted, [order, *ops[1:]], [x, ops[1].t().contiguous().t(), *ops[2:]]):
        for a, b in zip(_run(other, dy, "silu"), base):
            assert torch.equal(a, b)
    for strided in (dy.transpose(0, 1).contiguous().transpose(0, 1), dy[..., :1].expand(dy.shape), torch.cat([dy.flatten()[:1], dy.flatten()])[1:].view(dy.shape)):
        for a, b in zip(_run(ops, strided, "silu"), _run(ops, strided.clone(memory_format=torch.contiguous_format), "silu")):
            assert torch.equal(a, b)


def test_no_tokens():
    ops, dy = _operands(0, 64, 72, 80, F16, True)
    got = _run(ops, dy, "silu")
    assert got[0].shape == (0, 80) and got[1].shape == (0, 64)
    assert all(not g.any() for g in got[2:])


def test_extreme_values():
    """Gates of +-30000 and of zero, an infinite and a NaN row: what is finite stays exact, and nothing reaches another row."""
    for rows in (16, 300):
        ops, dy = _operands(rows, 64, 72, 80, BF16, False, seed=9)
        x = ops[0].clone()
        x[3], x[4], x[5], x[7] = 1e4, -1e4, 0.0, 1e-30
        clean = _run([x, *ops[1:]], dy, "silu")
        want = _exact([x, *ops[1:]], dy, "silu")
        for a, b in zip(clean[:2], want[:2]):  # row by row: their sizes differ by orders of magnitude
            for r in (0, 3, 4, 5, 7):
                assert _off(a[r], b[r]) < 2 * _bound(BF16) or b[r].norm() < 1e-25
        x[3], x[4] = float("nan"), float("inf")
        bad = _run([x, *ops[1:]], dy, "silu")
        keep = torch.ones(rows, dtype=torch.bool)
        keep[[3, 4]] = False
        assert torch.equal(bad[0][keep], clean[0][keep]) and torch.equal(bad[1][keep], clean[1][keep])
        assert bad[0][3].isnan().all()


def test_same_bits_every_time():
    ops, dy = _operands(2000, 256, 520, 264, BF16, True, seed=10)
    first = _run(ops, dy, "silu")
    for _ in range(3):
        for a, b in zip(_run(ops, dy, "silu"), first):
            assert torch.equal(a, b)


def test_rows_behind_the_last_are_left_alone():
    for rows in (5, 130):
        ops, _ = _operands(rows, 64, 72, 80, BF16, True)
        out = [torch.full((rows + 200, n), 7.0, dtype=BF16, device="cuda") for n in (80, 72)]
        size = _lib.lib().mf_gated_mlp_pre_bytes(rows, 72)
        pre = torch.full((size + 5000,), 77, dtype=torch.uint8, device="cuda")
        a = gated._args(*ops, "silu", BF16)
        a.y, a.act, a.pre = (t.data_ptr() for t in (*out, pre))
        _lib.launch(_lib.lib().mf_gated_mlp_fwd, ops[0].device, ctypes.byref(a))
        assert torch.equal(out[0][:rows], mfb.gated_mlp(*ops))
        assert all((t[rows:] == 7.0).all() for t in out) and (pre[size:] == 77).all()


def test_other_stream():
    ops, dy = _operands(500, 128, 264, 136, BF16, True, seed=11)
    want = _run(ops, dy, "silu")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.cuda._sleep(2_000_000)
        later = [t + 0 for t in ops]  # made on this stream, late
        got = _run(later, dy, "silu")
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows", [20, 300])
def test_captured_passes(rows):
    """Two graphs of forward and backward, replayed in turn on new data.  While an eager graph of the same leaves is alive the capture is refused."""
    first, dy = _operands(rows, 64, 136, 72, BF16, True, seed=12)
    second, _ = _operands(rows, 64, 136, 72, BF16, True, seed=13)
    want = [_run(first, dy, "silu"), _run(second, dy, "silu")]
    static = [t.clone().requires_grad_() for t in first]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            torch.autograd.grad(mfb.gated_mlp(*static), static, dy)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    alive = mfb.gated_mlp(*static)
    for params in (static[1:], [t.detach().float() for t in static[1:]]):  # both host paths
        with pytest.raises(RuntimeError, match="release that graph"), torch.cuda.graph(torch.cuda.CUDAGraph()):
            y = mfb.gated_mlp(static[0], *params)
            torch.autograd.grad(y, static[0], dy)
    del alive, y
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = mfb.gated_mlp(*static)
            outs.append([y.detach(), *torch.autograd.grad(y, static, dy)])
        graphs.append(graph)
    for values, expected in ((first, want[0]), (second, want[1]), (first, want[0])):
        with torch.no_grad():
            for t, v in zip(static, values):
                t.copy_(v)
        for graph, out in zip(graphs, outs):
            graph.replay()
            for a, b in zip(out, expected):
                assert torch.equal(a, b)


def test_two_host_threads():
    """Calls of different sizes from two threads, each on a stream of its own."""
    jobs = [_operands(rows, 64, F, 80, BF16, True, seed=20 + i) for i, (rows, F) in enumerate(((300, 72), (3000, 264)))]
    want = [_run(*job, "silu") for job in jobs]
    torch.cuda.synchronize()
    failures = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                if not all(torch.equal(a, b) for a, b in zip(_run(*jobs[i], "silu"), want[i])):
                    failures.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures


def test_once_differentiable():
    ops, dy = _operands(40, 64, 72, 80, BF16, True)
    for x in (ops[0], ops[0].repeat(1, 2)[:, :64]):  # both host paths
        x = x.detach().requires_grad_()
        (g,) = torch.autograd.grad(mfb.gated_mlp(x, *ops[1:]), x, dy, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.float().sum().backward()


def test_inputs_changed_in_place_are_noticed():
    ops, dy = _operands(40, 64, 72, 80, BF16, True)
    leaves = [t.detach().requires_grad_() for t in ops]
    y = mfb.gated_mlp(*leaves)
    with torch.no_grad():
        leaves[1].mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, leaves[0], dy)


@pytest.mark.parametrize("backward,kind", [(b, k) for b in (0, 1) for k in range(4)])
def test_expired_waits(backward, kind):
    """Hand-offs of one kind withheld: every wait ends at its limit, the call reports it, and the next call is whole.  Sizes with more
    blocks than stages and more tiles than accumulators for every pair of CTAs, so that each kind is waited for."""
    ops, dy = _operands(20000, 512, 520, 520, BF16, False, seed=14)
    want = _run(ops, dy, "silu")
    rows, F = ops[0].shape[0], 520
    a = gated._args(*ops, "silu", BF16)
    made = [torch.empty(_lib.lib().mf_gated_mlp_pre_bytes(rows, F), dtype=torch.uint8, device="cuda")]
    made += [torch.empty(rows, n, dtype=BF16, device="cuda") for n in (F, 520, 512)] + [torch.empty_like(t) for t in ops[1:3]]
    a.pre, a.act, a.y, a.grad_x, a.grad_w_in, a.grad_w_out = (t.data_ptr() for t in made)
    a.grad_y = dy.data_ptr()
    _lib.launch(_lib.lib().mf_gated_mlp_fwd, dy.device, ctypes.byref(a))
    need = _lib.lib().mf_gated_mlp_bwd_workspace_bytes(ctypes.byref(a))
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = ws.data_ptr(), need
    status = ctypes.c_int32(0)
    _lib.launch(_lib.lib().mf_selftest_gated_mlp_give_up, dy.device, ctypes.byref(a), backward, kind, 40000, ctypes.byref(status))
    assert status.value == _lib.MF_ERR_DEVICE_TIMEOUT
    assert mfb.gated_mlp_status() == 0
    for g, b in zip(_run(ops, dy, "silu"), want):
        assert torch.equal(g, b)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("rows", [20, 300])
def test_pre_activations_of_different_sizes(rows, dtype):
    """Tokens and channels whose pre-activations span many orders: each token's gradients against its own size.  The kept form goes by
    the largest of 16 channels, so a channel a thousand times smaller than its neighbour still has what the block's type gives it.

    Hidden values are products of two pre-activations and have to lie in the block's type: fp16 ends at 65504, so its factors stop at 2 and 8
    (pre-activations to 16 * 5 standard deviations, products to 6400), where bf16 takes 16 and 32."""
    g = torch.Generator().manual_seed(30)
    ops, dy = _operands(rows, 64, 80, 72, dtype, False, seed=31)
    ops[0] *= (2.0 ** torch.randint(-12, 5 if dtype == BF16 else 2, (rows, 1), generator=g)).to(dtype).cuda()
    ops[1] *= (2.0 ** torch.randint(-5, 6 if dtype == BF16 else 4, (160, 1), generator=g)).to(dtype).cuda()
    got, want = _run(ops, dy, "silu"), _exact(ops, dy, "silu")
    tiny = torch.finfo(dtype).tiny * 64  # fp16 has no more bits there
    for a, b in zip(got, want):
        size = b.norm(dim=1, keepdim=True) / b.shape[1] ** 0.5
        off = (a.double() - b).norm(dim=1) / (size.squeeze(1) * b.shape[1] ** 0.5).clamp_min(1e-300)
        assert (off[size.squeeze(1) > tiny] < 2 * _bound(dtype)).all()


@pytest.mark.parametrize("rows", [7, 33, 300])
def test_infinite_weight_and_the_rows_behind_the_last(rows):
    """An infinite weight makes its channel's gradients infinite; the tile's rows behind the last token, where it meets zeros, add nothing."""
    ops, dy = _operands(rows, 64, 72, 80, BF16, True, seed=40)
    ops[1] *= 0.01
    ops[3].fill_(2.0)  # positive pre-activations and slopes
    dy = dy.abs() + 0.1
    leaves = [t.detach().requires_grad_(i == 3) for i, t in enumerate(ops)]
    clean = torch.autograd.grad(mfb.gated_mlp(*leaves), leaves[3], dy)[0]
    leaves[2].data[0, 5] = float("inf")
    got = torch.autograd.grad(mfb.gated_mlp(*leaves), leaves[3], dy)[0]
    assert got[5] == got[72 + 5] == float("inf")
    others = torch.ones(144, dtype=torch.bool)
    others[[5, 77]] = False
    assert torch.equal(got[others], clean[others])


def test_widths_beyond_the_kernel_are_refused():
    wide, w = torch.zeros(1, 1, dtype=BF16, device="cuda").expand(1, 2**32 + 8), torch.zeros(8, 8, dtype=BF16, device="cuda")
    assert not gated.gated_mlp_applies(wide, wide.expand(16, -1), w)
    with pytest.raises(ValueError, match="up to 2\\^28"):
        mfb.gated_mlp(wide, wide.expand(16, -1), w)


def test_inference_mode():
    for rows in (5, 300):
        ops, _ = _operands(rows, 64, 72, 80, BF16, True, seed=41)
        want = mfb.gated_mlp(*ops)
        with torch.inference_mode():
            got = mfb.gated_mlp(*ops)
            assert got.is_inference() and torch.equal(got, want)


@pytest.mark.parametrize("rows", [1, 16, 32])
def test_weights_that_the_call_before_makes(rows):
    """Each call's result is the next call's output weight, without a pause between them: no kernel may read it too soon."""
    g = torch.Generator().manual_seed(42)
    x, xs = _randn(g, rows, 64), [_randn(g, 16, 64) for _ in range(100)]
    w_in, w_weight = _randn(g, 1024, 64) / 8, _randn(g, 512, 512) / 16  # (16, 64) -> a weight (16, 512) of 512 hidden channels
    weights = [mfb.gated_mlp(t, w_in, w_weight) for t in xs]
    torch.cuda.synchronize()
    want = []
    for w in weights:
        want.append(mfb.gated_mlp(x, w_in, w))
        torch.cuda.synchronize()
    buffer = torch.zeros(16, 512, dtype=BF16, device="cuda")
    a = gated._args(xs[0], w_in, w_weight, None, None, "silu", BF16)
    act, made = torch.empty(16, 512, dtype=BF16, device="cuda"), []
    a.act, a.y = act.data_ptr(), buffer.data_ptr()
    for t in xs:  # always into the same weight
        a.x = t.data_ptr()
        _lib.launch(_lib.lib().mf_gated_mlp_fwd, x.device, ctypes.byref(a))
        made.append(mfb.gated_mlp(x, w_in, buffer))
    for got, w in zip(made, want):
        assert torch.equal(got, w)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g).to(BF16).cuda()


@pytest.mark.parametrize("kind", range(3))
def test_expired_waits_in_narrow_tiles(kind):
    """The same for an output product that is a single round of narrow tiles over more blocks than stages (600 x 520 over 648)."""
    ops, _ = _operands(600, 64, 648, 520, BF16, True, seed=43)
    want = mfb.gated_mlp(*ops)
    a = gated._args(*ops, "silu", BF16)
    act, y = torch.empty(600, 648, dtype=BF16, device="cuda"), torch.empty(600, 520, dtype=BF16, device="cuda")
    a.act, a.y = act.data_ptr(), y.data_ptr()
    status = ctypes.c_int32(0)
    _lib.launch(_lib.lib().mf_selftest_gated_mlp_give_up, y.device, ctypes.byref(a), 0, kind, 40000, ctypes.byref(status))
    assert status.value == _lib.MF_ERR_DEVICE_TIMEOUT
    assert mfb.gated_mlp_status() == 0
    assert torch.equal(mfb.gated_mlp(*ops), want)
