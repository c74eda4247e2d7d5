"""Dense attention as programs use it: in layers, trunks and models, captured, on other streams, under transforms; expired waits."""
import copy
import ctypes

import pytest
import torch

import matterformer_b200 as mfb
from matterformer_b200 import _lib, dense
from matterformer_b200.dense import dense_attention_torch
from matterformer_b200.dp import GraphedTrainStep
from matterformer_b200.dp import GraphedTrainStep, edm_train_step
from matterformer_b200.trunk import EDMLoss, EDMModel, EDMPreconditioner, RegularAttention, TransformerTrunk

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _suffix(B, N):
    n = torch.linspace(N, max(1, N // 4), B, device="cuda").long()
    return torch.arange(N, device="cuda") >= n[:, None]


@pytest.mark.parametrize("holes", [False, True])
@pytest.mark.parametrize("heads,N", [(8, 29), (8, 181), (4, 300)])
def test_layer_against_the_library(heads, N, holes):
    """``impl="cuda"`` under bf16 autocast against nn.MultiheadAttention in fp32: 2e-2 of the largest value, as the other cores."""
    g = torch.Generator(device="cuda").manual_seed(N)
    layer = RegularAttention(512, heads, impl="cuda").cuda()
    plain = RegularAttention(512, heads, impl="torch").cuda()
    plain.load_state_dict(layer.state_dict())
    x, mask = _randn(g, 3, N, 512), _suffix(3, N)
    if holes:
        mask = torch.rand(3, N, generator=g, device="cuda") < 0.3
        mask[:, 0] = False
    grad = _randn(g, 3, N, 512) * ~mask[..., None]
    outs, grads = [], []
    for net, low in ((layer, True), (plain, False)):
        xi = x.clone().requires_grad_()
        with torch.autocast("cuda", BF16, enabled=low):
            out = net(xi, key_padding_mask=mask)
        outs.append(out.float())
        grads.append(torch.autograd.grad(out, [xi, *net.parameters()], grad.to(out.dtype)))
    assert layer._last_core_used == "dense"
    assert (outs[0] - outs[1])[~mask].abs().max() <= 2e-2 * outs[1].abs().max()
    for a, b in zip(*grads):
        assert (a.float() - b).abs().max() <= 2e-2 * b.abs().max()


@pytest.mark.parametrize("kind", ["distance", "offset"])
@pytest.mark.parametrize("N", [29, 150])
def test_biased_layer_against_plain_operations(N, kind):
    g = torch.Generator(device="cuda").manual_seed(N)
    spec = mfb.RelativeBias(32, kind, 8)
    layer = RegularAttention(256, 4, relative_bias=spec, rotary=mfb.RotaryPositions(48, axes=3)).cuda()
    torch.nn.init.normal_(layer.bias_table)
    plain = copy.deepcopy(layer)
    plain.impl = "torch"
    x, mask, coords = _randn(g, 4, N, 256), _suffix(4, N), _randn(g, 4, N, 3) * 3
    buckets = spec.buckets(coords, (~mask).sum(1), x.device)
    grad = _randn(g, 4, N, 256) * ~mask[..., None]
    results = []
    for net, low in ((layer, True), (plain, False)):
        with torch.autocast("cuda", BF16, enabled=low):
            out = net(x, key_padding_mask=mask, buckets=buckets, positions=coords)
        results.append((out.float()[~mask], *torch.autograd.grad(out, list(net.parameters()), grad.to(out.dtype))))
    assert (layer._last_core_used, plain._last_core_used) == ("dense", "torch")
    for a, b in zip(*results):
        assert (a.float() - b).abs().max() <= 2e-2 * b.abs().max()


def _model(**more):
    torch.manual_seed(0)
    model = EDMModel(d_model=256, n_heads=4, n_layers=4, **more).cuda()
    for block in model.trunk.blocks:
        torch.nn.init.normal_(block.ada_ln[-1].bias, std=0.2)
        torch.nn.init.normal_(block.ada_ln[-1].weight, std=0.02)
    return model


def _batch(B, N, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    mask = _suffix(B, N)
    return torch.randint(0, 5, (B, N), generator=g, device="cuda"), _randn(g, B, N, 3) * 2, mask, torch.rand(B, generator=g, device="cuda") + 0.2, \
        _randn(g, B, N, 6), _randn(g, B, N, 3)  # fmt: skip


@pytest.mark.parametrize("kind", ["distance", "offset"])
@pytest.mark.parametrize("N", [25, 60])
def test_training_step_of_a_model(N, kind):
    """Under bf16 autocast against the same model in fp32 plain operations; the tables move."""
    model = _model(relative_bias=mfb.RelativeBias(16, kind, 6))
    plain = copy.deepcopy(model)
    for block in plain.trunk.blocks:
        if isinstance(block.attn, RegularAttention):
            block.attn.impl = "torch"
    types, coords, mask, sigma, an, cn = _batch(6, N)
    losses = []
    for net, low in ((model, True), (plain, False)):
        with torch.autocast("cuda", BF16, enabled=low):
            loss, _ = EDMLoss()(EDMPreconditioner(net), types, coords, mask, sigma=sigma, atom_noise=an, coord_noise=cn)
        loss.backward()
        losses.append(float(loss.detach()))
    assert abs(losses[0] - losses[1]) <= 2e-2 * abs(losses[1])
    for a, b in zip(model.trunk.blocks, plain.trunk.blocks):
        if isinstance(a.attn, RegularAttention):
            assert a.attn._last_core_used == "dense"
            ga, gb = a.attn.bias_table.grad, b.attn.bias_table.grad
            assert (ga - gb).norm() <= 0.1 * gb.norm() and gb.norm() > 0


def test_captured_sampling_and_training():
    """Operators together, as a program has them: a captured denoiser with distances, gated blocks and rotary positions, equal to the eager one; a captured
    training step, whose parameters go the way of eager steps."""
    types, coords, mask, *_ = _batch(8, 29)
    more = {"relative_bias": mfb.RelativeBias(16, "distance", 6.0), "mlp_type": "gated", "rotary": mfb.RotaryPositions(48, axes=3)}
    net = EDMPreconditioner(_model(**more)).eval()
    g = torch.Generator(device="cuda").manual_seed(1)
    with torch.no_grad():
        den = mfb.GraphedDenoiser(net, _randn(g, 8, 29, 6), coords, mask, None, BF16)
        for sigma in (0.1, 1.0, 5.0):
            a, x = _randn(g, 8, 29, 6), _randn(g, 8, 29, 3)
            got = den(a, x, sigma)
            with torch.autocast("cuda", BF16):
                want = net(a, x, mask, torch.full((8,), sigma, device="cuda"))
            assert all(torch.equal(u, v.float()) for u, v in zip(got, want))
    for captured in (False, True):
        net = EDMPreconditioner(_model(**more))
        optimizer = torch.optim.AdamW(net.parameters(), lr=torch.tensor(1e-3), capturable=True)
        batch = {"atom_types": types, "coords": coords, "pad_mask": mask}
        torch.manual_seed(5)
        if captured:
            step = GraphedTrainStep(net, EDMLoss(), optimizer, batch, warmup=3)
        else:
            def step(net=net, optimizer=optimizer, batch=batch):
                return edm_train_step(net, EDMLoss(), optimizer, batch, autocast_dtype=BF16, clip=1.0)
        before = [b.attn.bias_table.detach().clone() for b in net.model.trunk.blocks if isinstance(b.attn, RegularAttention)]
        losses = [step().detach().clone() for _ in range(3)]
        torch.cuda.synchronize()
        after = [b.attn.bias_table for b in net.model.trunk.blocks if isinstance(b.attn, RegularAttention)]
        assert all(torch.isfinite(x) for x in losses) and all((u - v).abs().max() > 0 for u, v in zip(before, after))


def test_captured_passes_share_a_workspace_pool():
    """Two captured forward and backward passes that take their memory from one pool, replayed in turn on other data."""
    g = torch.Generator(device="cuda").manual_seed(0)
    calls = []
    for B, H, K, M, N, D in ((2, 4, 4, 300, 300, 64), (3, 8, 2, 2, 900, 128), (4, 2, 2, 29, 29, 64)):
        q, k, v = (_randn(g, *s).to(BF16).requires_grad_() for s in ((B, H, M, D), (B, K, N, D), (B, K, N, D)))
        table = _randn(g, 16, H).requires_grad_()
        buckets = mfb.offset_buckets(16, 30, device="cuda")
        grad = _randn(g, B, H, M, D).to(BF16)

        def step(q=q, k=k, v=v, table=table, buckets=buckets, grad=grad):
            out = mfb.dense_attention(q, k, v, bias=table, buckets=buckets, causal=True)
            return [out.detach(), *torch.autograd.grad(out, [q, k, v, table], grad)]

        calls.append((step, (q, k, v, table, grad)))
    stream, pool, graphs = torch.cuda.Stream(), None, []
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for step, _ in calls:
            step()
    torch.cuda.synchronize()
    for step, _ in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool, stream=stream):
            made = step()
        pool = graph.pool()
        graphs.append((graph, made))
    for _ in range(2):
        for (step, tensors), (graph, made) in zip(calls, graphs):
            with torch.no_grad():
                for t in tensors:
                    t.copy_(torch.randn_like(t))
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in made]
            with torch.cuda.stream(stream):
                want = step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams_at_once():
    g = torch.Generator(device="cuda").manual_seed(3)
    ops = [[_randn(g, 4, 8, 512, 64).to(BF16) for _ in range(3)] for _ in range(2)]
    table, buckets = _randn(g, 32, 8), mfb.offset_buckets(32, 64, device="cuda")

    def step(q, k, v):
        leaves = [t.detach().requires_grad_() for t in (q, k, v, table)]
        out = mfb.dense_attention(*leaves[:3], bias=leaves[3], buckets=buckets)
        return [out.detach(), *torch.autograd.grad(out, leaves, q)]

    want = [step(*o) for o in ops]
    streams = [torch.cuda.Stream() for _ in ops]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        got = []
        for s, o in zip(streams, ops):
            with torch.cuda.stream(s):
                got.append(step(*o))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_offsets_beyond_32_bits():
    """Entries that lie more than 2^31 elements apart."""
    far = 2**31 + 64 * 600
    store = torch.empty(far + 2 * 600 * 64, device="cuda", dtype=BF16)
    g = torch.Generator(device="cuda").manual_seed(0)
    for M, N in ((600, 600), (1, 600), (29, 29), (100, 100)):
        k = store.as_strided((2, 1, N, 64), (far, N * 64, 64, 1))
        small = _randn(g, 2, 1, N, 64).to(BF16)
        k.copy_(small)
        q = _randn(g, 2, 1, M, 64).to(BF16)
        assert torch.equal(mfb.dense_attention(q, k, k), mfb.dense_attention(q, small, small))
        leaves = [t.detach().requires_grad_() for t in (k, small)]
        ga, gb = (torch.autograd.grad(mfb.dense_attention(q, t, t).float().square().sum(), t)[0] for t in leaves)
        assert torch.equal(ga, gb)


def test_rows_behind_and_between_stay():
    """Results go to their rows alone: a strided result is not what the call makes, so the C interface is asked."""
    g = torch.Generator(device="cuda").manual_seed(0)
    B, H, N, D = 2, 2, 70, 64
    q, k, v = (_randn(g, B, H, N, D).to(BF16) for _ in range(3))
    wide = torch.full((B, H, N + 3, D + 8), 7.0, device="cuda", dtype=BF16)
    for backend in ("mma", "tcgen05"):
        prev = mfb.set_dense_backend(backend)
        a = dense._args(q, k, v, None, None, None, None, None, False, 0.125)
        wide.fill_(7.0)
        a.out, a.out_rows = wide.data_ptr(), _lib.MfRows(wide.stride(0), wide.stride(1), wide.stride(2))
        _lib.launch(_lib.lib().mf_dense_attn_fwd, q.device, ctypes.byref(a))
        want = mfb.dense_attention(q, k, v)
        mfb.set_dense_backend(prev)
        assert torch.equal(wide[:, :, :N, :D], want) and (wide[:, :, N:] == 7).all() and (wide[:, :, :, D:] == 7).all()


def test_transforms_and_traces():
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (_randn(g, 2, 2, 40, 32).half() for _ in range(3))
    table, buckets = _randn(g, 8, 2), mfb.offset_buckets(8, 10, device="cuda")
    want = dense_attention_torch(q, k, v, bias=table, buckets=buckets)
    many = torch.func.vmap(lambda t: mfb.dense_attention(q, k, v, bias=t, buckets=buckets))(torch.stack([table, table]))
    assert torch.equal(many[1], want)
    out, tangent = torch.func.jvp(lambda t: mfb.dense_attention(t, k, v, bias=table, buckets=buckets), (q,), (torch.ones_like(q),))
    assert torch.equal(out, want) and torch.isfinite(tangent).all()
    traced = torch.jit.trace(lambda a, b, c: mfb.dense_attention(a, b, c, bias=table, buckets=buckets), (q, k, v))
    assert torch.equal(traced(k, q, v), dense_attention_torch(k, q, v, bias=table, buckets=buckets))


def test_autograd_rules():
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (_randn(g, 1, 2, 40, 64).to(BF16).requires_grad_() for _ in range(3))
    out = mfb.dense_attention(q, k, v)
    grad = torch.autograd.grad(out.float().sum(), q, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="differentiate twice"):
        grad.float().sum().backward()
    out = mfb.dense_attention(q, k, v)
    with torch.no_grad():
        k.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    with torch.inference_mode():
        counts, mask = torch.tensor([30], device="cuda", dtype=torch.int32), torch.ones(1, 40, dtype=torch.bool, device="cuda")
    mfb.dense_attention(q, k, v, counts, counts, key_mask=mask).sum().backward()


@pytest.mark.parametrize("change,message", [
    ({"k": (1, 3, 40, 64)}, "multiple of K"), ({"v": (1, 2, 41, 64)}, "expected"), ({"dim": 48}, "head_dim"), ({"dtype": torch.float32}, "only supports"),
    ({"bias": (8, 2)}, "go together"), ({"bias": (129, 2), "buckets": (5,)}, "up to 128"), ({"bias": (8, 3), "buckets": (5,)}, "bias"),
    ({"bias": (8, 2), "buckets": (6,)}, "buckets"), ({"bias": (8, 2), "buckets": (2, 40, 40)}, "buckets"), ({"key_mask": (1, 39)}, "key_mask"),
    ({"num_keys": 2}, "num_keys"), ({"scale": float("nan")}, "scale"),
])  # fmt: skip
def test_refusals_on_the_gpu(change, message):
    dim, dtype = change.get("dim", 64), change.get("dtype", BF16)
    z = lambda *s, **o: torch.zeros(*s, device="cuda", **o)  # noqa: E731
    q, k, v = (z(*change.get(n, (1, 2, 40, dim)), dtype=dtype) for n in "qkv")
    more = {}
    if "bias" in change:
        more["bias"] = z(*change["bias"])
    if "buckets" in change:
        more["buckets"] = z(*change["buckets"], dtype=torch.uint8)
    if "key_mask" in change:
        more["key_mask"] = z(*change["key_mask"], dtype=torch.bool)
    if "num_keys" in change:
        more["num_keys"] = z(change["num_keys"], dtype=torch.int32)
    if "scale" in change:
        more["scale"] = change["scale"]
    with pytest.raises((ValueError, RuntimeError), match=message):
        mfb.dense_attention(q, k, v, **more)


def _expire(backward, kind, host_status, head_dim=64):
    """A call of 200 queries on 900 of 1000 keys, more tiles than buffers, with the hand-offs of one kind withheld."""
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v, out, go = (_randn(g, 1, 2, n, head_dim).to(BF16) for n in (200, 1000, 1000, 200, 200))
    num = torch.tensor([900], device="cuda", dtype=torch.int32)
    lse = torch.zeros(1, 2, 200, device="cuda")
    prev = mfb.set_dense_backend("tcgen05")
    a = dense._args(q, k, v, None, num, None, None, None, False, 0.125)
    mfb.set_dense_backend(prev)
    a.out, a.out_rows, a.lse, a.grad_out, a.grad_out_rows = out.data_ptr(), dense._rows(out), lse.data_ptr(), go.data_ptr(), dense._rows(go)
    grads = [torch.empty_like(t) for t in (q, k, v)]
    for name, t in zip(("dq", "dk", "dv"), grads):
        setattr(a, name, t.data_ptr())
        setattr(a, name + "_rows", dense._rows(t))
    ws = dense._workspace(a, _lib.lib().mf_dense_attn_bwd_workspace_bytes(ctypes.byref(a)), q.device)  # noqa: F841
    _lib.launch(_lib.lib().mf_selftest_dense_attn_give_up, q.device, ctypes.byref(a), int(backward), kind, 40000, host_status)
    torch.cuda.synchronize()


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("kind", range(5))
@pytest.mark.parametrize("backward", [False, True])
def test_expired_waits_end_and_are_told(backward, kind, head_dim):
    status = ctypes.c_int32(0)
    _expire(backward, kind, ctypes.byref(status), head_dim)
    assert status.value == _lib.MF_ERR_DEVICE_TIMEOUT
    assert mfb.dense_attention_status() == 0  # the self-test keeps it to itself
    q = torch.randn(1, 2, 300, head_dim, device="cuda").to(BF16)
    assert torch.isfinite(mfb.dense_attention(q, q, q)).all() and mfb.dense_attention_status() == 0


def test_checked_calls_raise():
    _expire(False, 0, None)
    assert mfb.dense_attention_status() == _lib.MF_ERR_DEVICE_TIMEOUT and mfb.dense_attention_status() == 0
    previous = mfb.set_check_status(True)
    try:
        q = torch.randn(1, 2, 300, 64, device="cuda").to(BF16).requires_grad_()
        out = mfb.dense_attention(q, q, q)
        _expire(True, 0, None)
        with pytest.raises(RuntimeError, match="expired"):
            out.sum().backward()
        mfb.dense_attention(q, q, q).sum().backward()
        _expire(False, 2, None)
        with pytest.raises(RuntimeError, match="expired"):
            mfb.dense_attention(q, q, q)
    finally:
        mfb.set_check_status(previous)
