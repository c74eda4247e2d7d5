"""Dense attention with a learned bias by buckets, and distance buckets, against their definitions in 64 bits.

Tolerances: with u half a step of the operands' type (2^-8 bf16, 2^-11 fp16), p off by at most u p where it enters a product and a result by u
of itself, so |out - exact| <= u (p |v|) + u |out|; delta = grad . out takes out's error over; dS = p (dP - delta) is rounded once more.  fp32: logits of
magnitude z are off by some z 2^-22, and p by that in relation, sums by n 2^-24 at most; `slack` stands for both.  Small p: the exponential gives zero
below 2^-126, and in fp16 a probability or a gradient of a logit below 2^-14 is off by up to 2^-25 whatever its size; `floor` is that error of
one entry, absolute, and enters each sum once for every entry (a gradient of a logit that comes from such a p with the factor |dP| + |delta|).
"""
import math

import pytest
import torch

import matterformer_b200 as mfb
from matterformer_b200.dense import dense_attention_torch

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def exact(q, k, v, grad, num_keys, num_queries, key_mask, causal, bias, buckets, scale):
    """Output, gradients and their bounds, fp64: a dict name -> (value, bound)."""
    u = torch.finfo(q.dtype).eps / 2
    B, H, M, D = q.shape
    K, N = k.shape[1:3]
    G = H // K
    dev = q.device
    i, j = torch.arange(M, device=dev)[:, None], torch.arange(N, device=dev)
    nq = torch.full((B, 1, 1), M, device=dev) if num_queries is None else num_queries.long().view(B, 1, 1)
    nk = torch.full((B, 1, 1), N, device=dev) if num_keys is None else num_keys.long().view(B, 1, 1)
    off = j - i - (nk - nq)
    see = (i < nq) & (j < nk)
    if causal:
        see = see & (off <= 0)
    if key_mask is not None:
        see = see & key_mask[:, None]
    see = see.expand(B, M, N)[:, None]
    qd, kd, vd = q.double(), k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    qd = torch.where(see.any(3)[..., None], qd, 0.0)
    kd, vd = (torch.where(see.any(2)[..., None], t, 0.0) for t in (kd, vd))
    z = scale * qd @ kd.transpose(-1, -2)
    if bias is not None:
        if buckets.ndim == 1:
            L = buckets.numel() // 2
            which = buckets[off.clamp(-L, L) + L].long().expand(B, M, N)
        else:
            which = buckets.long().expand(B, M, N)
        inside = which < bias.shape[0]
        value = torch.where(inside[..., None], bias.double()[which.clamp(max=bias.shape[0] - 1)], 0.0).permute(0, 3, 1, 2)
        see = see & ~(value < -1e30)
        z = z + torch.where(see, value, 0.0)
    z = torch.where(see, z, -math.inf)
    top = z.max(-1, keepdim=True).values
    p = torch.exp(z - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    reach = z.masked_fill(~see, 0.0).abs().max().item()
    slack = (1 + reach) * 2.0**-20 + N * 2.0**-24
    tiny = torch.finfo(q.dtype).tiny
    floor = 2.0**-126 if q.dtype == torch.bfloat16 else 2.0**-25
    out = p @ vd
    e_out = (u + slack) * (p @ vd.abs()) + u * out.abs() + tiny
    res = {"out": (out, e_out)}
    if grad is None:
        return res
    gd = torch.where((i < nq)[:, None, :, :1].expand(B, 1, M, 1), grad.double(), 0.0)
    dp = gd @ vd.transpose(-1, -2)
    delta = (gd * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_delta = (gd.abs() * e_out).sum(-1, keepdim=True) + slack * (gd.abs() * out.abs()).sum(-1, keepdim=True)
    e_ds = p * e_delta + slack * p * ((gd.abs() @ vd.abs().transpose(-1, -2)) + delta.abs())
    step = u * ds.abs() + e_ds + floor + 2.0**-126 * (dp.abs() + delta.abs())
    sc = abs(scale)

    def shared(t):
        return t.view(B, K, G, N, D).sum(2)

    dq, dk, dv = scale * ds @ kd, scale * shared(ds.transpose(-1, -2) @ qd), shared(p.transpose(-1, -2) @ gd)
    long = G * M * 2.0**-24
    res["dq"] = dq, sc * (step + N * 2.0**-24 * ds.abs()) @ kd.abs() + u * dq.abs() + tiny
    res["dk"] = dk, sc * shared((step + long * ds.abs()).transpose(-1, -2) @ qd.abs()) + u * dk.abs() + tiny
    res["dv"] = dv, shared(((u + slack + long) * p + floor).transpose(-1, -2) @ gd.abs()) + u * dv.abs() + tiny
    if bias is not None:
        nb = bias.shape[0]
        inside = inside[:, None].expand_as(ds)
        at = which[:, None].expand_as(ds).clamp(max=nb - 1)
        sums = []
        for t in (ds, e_ds + 2.0**-20 * ds.abs()):
            t = torch.where(inside, t, 0.0)
            sums.append(torch.stack([torch.zeros(nb, dtype=torch.float64, device=dev).index_add(0, at[:, h].reshape(-1), t[:, h].reshape(-1)) for h in range(H)], 1))
        res["dbias"] = sums[0], sums[1] + torch.finfo(bias.dtype).eps / 2 * sums[0].abs() + 1e-30
    return res


def check(got, want):
    for name, (value, bound) in want.items():
        g = got[name].double()
        assert torch.isfinite(g).all(), name
        over = ((g - value).abs() / bound).max().item() if g.numel() else 0.0
        assert over <= 1.0, (name, over)


def operands(seed, B, H, K, M, N, D, dtype, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return g, (spread * rnd(B, H, M, D)).to(dtype), rnd(B, K, N, D).to(dtype), rnd(B, K, N, D).to(dtype), rnd(B, H, M, D).to(dtype)


def run_both(q, k, v, grad, num_keys=None, num_queries=None, key_mask=None, causal=False, bias=None, buckets=None, scale=None):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)] + ([bias.detach().requires_grad_()] if bias is not None else [])
    out = mfb.dense_attention(*leaves[:3], num_keys, num_queries, key_mask=key_mask, causal=causal, bias=leaves[3] if bias is not None else None, buckets=buckets,
                              scale=scale)  # fmt: skip
    grads = torch.autograd.grad(out, leaves, grad)
    got = dict(zip(("out", "dq", "dk", "dv", "dbias"), (out.detach(), *grads)))
    sc = q.shape[-1] ** -0.5 if scale is None else scale
    want = exact(q, k, v, grad, num_keys, num_queries, key_mask, causal, bias, buckets, sc)
    check(got, want)
    with torch.no_grad():  # the call without gradients is the same
        assert torch.equal(got["out"], mfb.dense_attention(q, k, v, num_keys, num_queries, key_mask=key_mask, causal=causal, bias=bias, buckets=buckets, scale=scale))
    return got


@pytest.fixture(autouse=True, params=["auto", "mma", "tcgen05"])
def backend(request):
    """Every test on every family of kernels."""
    prev = mfb.set_dense_backend(request.param)
    yield
    mfb.set_dense_backend(prev)


def counts(g, B, most):
    n = torch.randint(0, most + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    n[0] = most
    return n


SIZES = [  # B, H, K, M, N
    (1, 1, 1, 1, 1), (3, 2, 2, 5, 5), (4, 8, 8, 29, 29), (2, 4, 2, 32, 32), (2, 2, 1, 33, 31), (3, 4, 4, 64, 64), (2, 4, 1, 65, 129), (1, 2, 2, 127, 128),
    (2, 3, 3, 181, 181), (1, 2, 1, 300, 257), (1, 2, 2, 515, 700), (2, 8, 2, 1, 777), (1, 4, 1, 3, 1025)]  # fmt: skip


@pytest.mark.parametrize("bias", ["none", "offset", "pair"])
@pytest.mark.parametrize("D,dtype", [(64, "bf16"), (32, "f16"), (128, "bf16"), (128, "f16"), (64, "f16")])
@pytest.mark.parametrize("B,H,K,M,N", SIZES)
def test_values_and_gradients(B, H, K, M, N, D, dtype, bias):
    g, q, k, v, grad = operands(M * 1000 + N + D, B, H, K, M, N, D, TYPES[dtype])
    table = buckets = None
    if bias != "none":
        nb = 16 if bias == "offset" else 21
        table = torch.randn(nb, H, generator=g, device="cuda").to(torch.float32 if D == 64 else TYPES[dtype])
        buckets = mfb.offset_buckets(nb, 40, device="cuda") if bias == "offset" else torch.randint(0, nb, (B, M, N), generator=g, device="cuda", dtype=torch.uint8)
    run_both(q, k, v, grad, bias=table, buckets=buckets)


@pytest.mark.parametrize("bias", ["none", "offset", "pair"])
@pytest.mark.parametrize("mask", ["lengths", "causal", "holes", "all"])
@pytest.mark.parametrize("B,H,K,M,N,D", [(5, 2, 2, 29, 29, 64), (4, 4, 2, 100, 100, 64), (3, 4, 1, 181, 300, 128), (3, 2, 2, 17, 40, 32), (4, 8, 2, 1, 500, 128),
                                         (2, 2, 1, 400, 260, 64), (2, 2, 1, 700, 700, 128)])  # fmt: skip
def test_masks(B, H, K, M, N, D, mask, bias):
    """Lengths down to nothing, causal calls with more queries than keys among them, masks with rows that leave nothing; garbage in hidden places."""
    g, q, k, v, grad = operands(M + N + D, B, H, K, M, N, D, torch.bfloat16)
    num_k = counts(g, B, N) if mask in ("lengths", "all") else None
    num_q = counts(g, B, M) if mask in ("lengths", "all") else None
    if num_k is not None:
        num_k[-1] = 0
    key_mask = None
    if mask in ("holes", "all"):
        key_mask = torch.rand(B, N, generator=g, device="cuda") < 0.7
        key_mask[-1] = False
        key_mask[0, : N // 2] = False
    for b in range(B):
        hidden = torch.zeros(N, dtype=torch.bool, device="cuda")
        if num_k is not None:
            hidden[num_k[b] :] = True
        if key_mask is not None:
            hidden |= ~key_mask[b]
        k[b, :, hidden], v[b, :, hidden] = float("nan"), float("inf")
        if num_q is not None:
            q[b, :, num_q[b] :], grad[b, :, num_q[b] :] = float("-inf"), float("nan")
    table = buckets = None
    if bias != "none":
        table = torch.randn(32, H, generator=g, device="cuda")
        table[3] = float("-inf")
        table[5, 0] = torch.finfo(torch.float32).min
        buckets = mfb.offset_buckets(32, 64, device="cuda") if bias == "offset" else torch.randint(0, 40, (1, M, N), generator=g, device="cuda", dtype=torch.uint8)
    got = run_both(q, k, v, grad, num_k, num_q, key_mask, mask in ("causal", "all"), table, buckets)
    if num_q is not None:
        for b in range(B):
            assert not got["out"][b, :, num_q[b] :].any() and not got["dq"][b, :, num_q[b] :].any()
            assert not got["dk"][b, :, num_k[b] :].any() and not got["dv"][b, :, num_k[b] :].any()


@pytest.mark.parametrize("M", [29, 181, 600])
def test_large_logits_and_one_key(M):
    """Sharp rows, where one key takes all, and rows of equal logits."""
    _, q, k, v, grad = operands(M, 2, 2, 2, M, M, 64, torch.bfloat16, spread=40.0)
    run_both(q, k, v, grad)
    run_both(torch.zeros_like(q), k, v, grad)
    run_both(q, k, v, grad, num_keys=torch.tensor([1, M], device="cuda", dtype=torch.int64), scale=-0.3)


@pytest.mark.parametrize("N", [29, 100, 400])
@pytest.mark.parametrize("heads,D", [(8, 64), (2, 128)])
def test_packed(N, heads, D):
    g = torch.Generator(device="cuda").manual_seed(N)
    B = 4
    qkv = torch.randn(B, N, 3 * heads * D, generator=g, device="cuda").bfloat16().requires_grad_()
    num = counts(g, B, N)
    coords = torch.randn(B, N, 3, generator=g, device="cuda") * 3
    buckets = mfb.distance_buckets(coords, torch.linspace(0, 8, 24)[1:], num)
    table = torch.randn(24, heads, generator=g, device="cuda").requires_grad_()
    grad = torch.randn(B, N, heads * D, generator=g, device="cuda").bfloat16()
    out = mfb.dense_attention_packed(qkv, heads, num, bias=table, buckets=buckets)
    dqkv, dtable = torch.autograd.grad(out, [qkv, table], grad)
    q, k, v = qkv.detach().view(B, N, 3, heads, D).permute(2, 0, 3, 1, 4)
    split = lambda t: t.view(B, N, heads, D).transpose(1, 2)  # noqa: E731
    want = exact(q, k, v, split(grad), num, num, None, False, table.detach(), buckets, D**-0.5)
    dq, dk, dv = dqkv.view(B, N, 3, heads, D).permute(2, 0, 3, 1, 4)
    check({"out": split(out), "dq": dq, "dk": dk, "dv": dv, "dbias": dtable}, want)


def test_strides_orders_and_offsets():
    """Token-major operands, every other head, a row that starts off a boundary, an expanded batch of keys and of buckets."""
    g, q, k, v, grad = operands(5, 3, 4, 2, 70, 90, 64, torch.float16)
    want = run_both(q, k, v, grad)
    tm = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    got = run_both(tm(q), tm(k), v, tm(grad))
    assert all(torch.equal(got[n], want[n]) for n in want) and got["out"].stride(1) == 64
    wide = torch.zeros(3, 8, 70, 72, device="cuda", dtype=torch.float16)
    wide[:, ::2, :, 3:67] = q
    got = run_both(wide[:, ::2, :, 3:67], k, v, grad)
    assert all(torch.equal(got[n], want[n]) for n in want)
    run_both(q, k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1), grad)
    table = torch.randn(5, 4, generator=g, device="cuda").half()
    pairs = torch.randint(0, 5, (90, 70), generator=g, device="cuda", dtype=torch.uint8)
    a = run_both(q, k, v, grad, bias=table, buckets=pairs.t())
    b = run_both(q, k, v, grad, bias=table, buckets=pairs.t().contiguous().expand(3, 70, 90))
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_repeatable_and_batch_independent():
    g, q, k, v, grad = operands(9, 6, 4, 4, 150, 150, 64, torch.bfloat16)
    table, buckets = torch.randn(32, 4, generator=g, device="cuda"), mfb.offset_buckets(32, 64, device="cuda")
    a = run_both(q, k, v, grad, bias=table, buckets=buckets)
    b = run_both(q, k, v, grad, bias=table, buckets=buckets)
    assert all(torch.equal(a[n], b[n]) for n in a)
    one = run_both(q[2:3], k[2:3], v[2:3], grad[2:3], bias=table, buckets=buckets)
    assert all(torch.equal(a[n][2:3], one[n]) for n in ("out", "dq", "dk", "dv"))


def test_gradient_against_differences():
    """The table's gradient and that of the operands along a direction, against differences of the plain form in 64 bits."""
    g, q, k, v, grad = operands(3, 2, 2, 1, 40, 52, 64, torch.float16)
    table, buckets = torch.randn(8, 2, generator=g, device="cuda"), torch.randint(0, 8, (2, 40, 52), generator=g, device="cuda", dtype=torch.uint8)
    got = run_both(q, k, v, grad, bias=table, buckets=buckets)
    ts = [t.double() for t in (q, k, v, table)]
    dirs = [torch.randn(t.shape, generator=g, device="cuda", dtype=torch.float64) for t in ts]
    f = lambda *x: (dense_attention_torch(*x[:3], bias=x[3], buckets=buckets) * grad.double()).sum()  # noqa: E731
    for i, name in enumerate(("dq", "dk", "dv", "dbias")):
        h = 1e-5
        plus, minus = ([t + s * h * d if n == i else t for n, (t, d) in enumerate(zip(ts, dirs))] for s in (1, -1))
        want = (f(*plus) - f(*minus)) / (2 * h)
        value, bound = exact(q, k, v, grad, None, None, None, False, table, buckets, 64**-0.5)[name]
        assert abs((got[name].double() * dirs[i]).sum() - want) <= (bound * dirs[i].abs()).sum() + 1e-6 * want.abs()
        assert abs((value * dirs[i]).sum() - want) <= 1e-6 * (value.abs() * dirs[i].abs()).sum()


def test_part_of_the_gradients_and_empty_calls():
    g, q, k, v, grad = operands(4, 2, 2, 2, 50, 50, 64, torch.bfloat16)
    table, buckets = torch.randn(8, 2, generator=g, device="cuda"), mfb.offset_buckets(8, 10, device="cuda")
    full = run_both(q, k, v, grad, bias=table, buckets=buckets)
    for name, i in (("dq", 0), ("dk", 1), ("dv", 2), ("dbias", 3)):
        args = [t.detach().clone() for t in (q, k, v, table)]
        args[i].requires_grad_()
        out = mfb.dense_attention(*args[:3], bias=args[3], buckets=buckets)
        assert torch.equal(torch.autograd.grad(out, args[i], grad)[0], full[name])
    for M, N, B in ((0, 50, 2), (50, 0, 2), (50, 50, 0), (0, 0, 1)):
        x, y = q[:B, :, :M].detach().requires_grad_(), k[:B, :, :N].detach().requires_grad_()
        t = table.detach().requires_grad_()
        out = mfb.dense_attention(x, y, y, bias=t, buckets=buckets)
        assert out.shape == (B, 2, M, 64) and not out.any()
        grads = torch.autograd.grad(out, [x, y, t], torch.ones_like(out))
        assert all(not g_.any() and g_.shape == like.shape for g_, like in zip(grads, (x, y, t)))


@pytest.mark.parametrize("B,N,edges", [(1, 1, 3), (3, 29, 31), (2, 200, 63), (1, 1000, 127), (5, 64, 0)])
def test_distance_buckets(B, N, edges):
    g = torch.Generator(device="cuda").manual_seed(N)
    x = torch.randn(B, N, 3, generator=g, device="cuda") * 4
    x[:, N // 2] = x[:, 0]  # two atoms in one place, distance exactly at an edge of zero
    num = counts(g, B, N)
    e = torch.linspace(0.0, 12.0, edges) if edges else torch.zeros(0)
    got = mfb.distance_buckets(x, e, num)
    d = (x.double()[:, :, None] - x.double()[:, None]).square().sum(-1)
    want = torch.zeros(B, N, N, dtype=torch.int64, device="cuda")
    for value in e.double().tolist():
        want += d >= value * value
    real = torch.arange(N, device="cuda") < num[:, None]
    want = torch.where(real[:, :, None] & real[:, None], want, 0)
    assert got.dtype == torch.uint8 and torch.equal(got.long(), want)
    assert torch.equal(mfb.distance_buckets(x, e.tolist(), num.long()), got) and torch.equal(mfb.distance_buckets(x.cpu(), e, num.cpu()), got.cpu())


@pytest.mark.parametrize("B,H,K,M,N,D", [(64, 8, 8, 5, 5, 64), (48, 8, 4, 33, 40, 128), (16, 8, 8, 100, 64, 64), (8, 4, 4, 130, 200, 64), (6, 4, 2, 90, 130, 128)])
@pytest.mark.parametrize("bias", ["none", "offset", "pair"])
def test_repeated_calls_are_bit_equal(B, H, K, M, N, D, bias):
    """Short walks, in which some warps of a block have no step of their own and run ahead of the rest: every sum has a fixed order, so that whatever
    differs between two calls was read before it was written, or written before it was read."""
    g, q, k, v, grad = operands(M + 7 * N, B, H, K, M, N, D, torch.bfloat16)
    table = buckets = None
    if bias != "none":
        table = torch.randn(16, H, generator=g, device="cuda")
        buckets = mfb.offset_buckets(16, 40, device="cuda") if bias == "offset" else torch.randint(0, 16, (B, M, N), generator=g, device="cuda", dtype=torch.uint8)
    first = run_both(q, k, v, grad, bias=table, buckets=buckets)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)] + ([table.requires_grad_()] if table is not None else [])
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(40):
        out = mfb.dense_attention(*leaves[:3], bias=table, buckets=buckets)
        made = [out.detach(), *torch.autograd.grad(out, leaves, grad)]
        for a, b in zip(made, first.values()):
            differ += (a != b).sum()
    assert int(differ) == 0


@pytest.mark.parametrize("M,N", [(29, 29), (3, 700), (150, 140), (300, 400)])
def test_broadcast_operands(request, M, N):
    """Keys of one head for all, one key for all places, one query for all: strides of zero, and their gradients before they are added up.
    Such operands run on the warp-level family where dense ones may run on tcgen05: equal bits are asked for where both run on one, the bounds always."""
    g, q, k, v, grad = operands(M + N, 2, 4, 2, M, N, 64, torch.bfloat16)
    table, buckets = torch.randn(16, 4, generator=g, device="cuda"), mfb.offset_buckets(16, 40, device="cuda")
    same = lambda t, d: t.narrow(d, 0, 1).expand_as(t)  # noqa: E731
    for x, y, z in ((q, same(k, 1), same(v, 1)), (same(q, 2), k, v), (q, same(k, 2), v), (same(q, 0), same(k, 0), same(v, 2))):
        got = run_both(x, y, z, grad, bias=table, buckets=buckets)
        if request.node.callspec.params["backend"] == "mma":
            dense = run_both(*(t.contiguous() for t in (x, y, z)), grad, bias=table, buckets=buckets)
            assert all(torch.equal(got[n], dense[n]) for n in got)
    leaf = k[:, :1].detach().clone().requires_grad_()
    out = mfb.dense_attention(q, leaf.expand_as(k), v, bias=table, buckets=buckets)
    made = torch.autograd.grad(out, leaf, grad)[0]
    whole = run_both(q, same(k, 1), v, grad, bias=table, buckets=buckets)["dk"]
    assert torch.equal(made, whole.sum(1, keepdim=True))


def test_distances_that_are_no_numbers():
    x = torch.randn(2, 70, 3, generator=torch.Generator().manual_seed(0)) * 3
    x[0, 5, 1], x[1, 0, 0], x[1, 40, 2], x[1, 41, 2] = float("nan"), float("inf"), -float("inf"), 3e38
    edges = torch.linspace(0.0, 12.0, 32, dtype=torch.float64)[1:]
    assert torch.equal(mfb.distance_buckets(x.cuda(), edges).cpu(), mfb.distance_buckets(x, edges))


@pytest.mark.parametrize("bias", ["none", "offset", "pair"])
@pytest.mark.parametrize("mask", ["none", "lengths", "causal", "holes"])
@pytest.mark.parametrize("B,H,K,M,N,D", [(1, 2, 1, 300, 2500, 128), (2, 3, 1, 270, 2111, 64), (3, 1, 1, 400, 4097, 64), (1, 4, 4, 130, 2048, 128), (1, 1, 1, 2600, 2600, 64)])
def test_few_tiles_of_queries_on_many_keys(B, H, K, M, N, D, mask, bias):
    """Keys in pieces on tiles of 128 queries: pieces that some rows see nothing of, or nobody does; rows without a key; garbage in hidden places."""
    g, q, k, v, grad = operands(M + N, B, H, K, M, N, D, torch.bfloat16)
    num_k = num_q = key_mask = None
    if mask == "lengths":
        num_k, num_q = counts(g, B, N), counts(g, B, M)
        num_k[-1] = N // 3 if B == 1 else 0
        num_q[0] = M - 1
        for b in range(B):
            k[b, :, num_k[b] :], v[b, :, num_k[b] :], q[b, :, num_q[b] :] = math.nan, math.inf, math.nan
    if mask == "holes":
        key_mask = torch.rand(B, N, generator=g, device="cuda") < 0.7
        key_mask[0, N // 4 : N // 4 + 1000] = False
        key_mask[-1, :700] = False
        for b in range(B):
            k[b, :, ~key_mask[b]], v[b, :, ~key_mask[b]] = math.nan, -math.inf
    table = buckets = None
    if bias != "none":
        table = torch.randn(16, H, generator=g, device="cuda")
        table[3, 0] = -math.inf
        buckets = mfb.offset_buckets(16, 40, device="cuda") if bias == "offset" else torch.randint(0, 18, (B, M, N), generator=g, device="cuda", dtype=torch.uint8)
    kw = dict(num_keys=num_k, num_queries=num_q, key_mask=key_mask, causal=mask == "causal", bias=table, buckets=buckets)
    with torch.no_grad():
        out = mfb.dense_attention(q, k, v, num_k, num_q, key_mask=key_mask, causal=mask == "causal", bias=table, buckets=buckets)
        check({"out": out}, exact(q, k, v, None, num_k, num_q, key_mask, mask == "causal", table, buckets, D**-0.5))
        again = mfb.dense_attention(q, k, v, num_k, num_q, key_mask=key_mask, causal=mask == "causal", bias=table, buckets=buckets)
        assert torch.equal(out, again)
    if N < 2600:  # the log-sum-exp that the backward pass reads
        run_both(q, k, v, grad, **kw)


def test_no_wait_expired_in_all_of_these():
    """Runs last: the status word gathers since it was last asked for."""
    assert mfb.dense_attention_status() == 0
