"""Dense attention and distance buckets where inputs are unusual: padding that is not at the end, values that are no numbers, empty calls, strides of
zero, many query heads on one key head."""
import copy
import math

import pytest
import torch
from test_dense_attention_gpu import counts, operands, run_both

import matterformer_b200 as mfb
from matterformer_b200 import _lib
from matterformer_b200.trunk import EDMModel, RegularAttention, TransformerTrunk

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
NAN = math.nan


@pytest.fixture
def backend(request):
    prev = mfb.set_dense_backend(request.param)
    yield request.param
    mfb.set_dense_backend(prev)


def _pad_masks(form, B, N):
    """Padding in front, in the middle, or at random places; every row keeps at least two atoms."""
    g = torch.Generator().manual_seed(N)
    if form == "front":
        return torch.arange(N) < torch.tensor([0, N // 3, N - 2])[:B, None]
    if form == "middle":
        return (torch.arange(N) >= N // 4) & (torch.arange(N) < N // 4 + torch.tensor([1, N // 3, N // 2])[:B, None])
    mask = torch.rand(B, N, generator=g) < 0.4
    mask[:, [0, N - 1]] = False
    return mask


@pytest.mark.parametrize("impl", ["auto", "torch"])
@pytest.mark.parametrize("form", ["front", "middle", "random"])
@pytest.mark.parametrize("N", [6, 29, 150])
def test_distances_beside_padding_anywhere(N, form, impl):
    """A trunk biased by distances: the buckets that its layers get are those of the distances for all pairs of atoms, and its output and the tables' gradients are
    those of the same trunk in fp32 on the CPU: within 1e-3 of the largest value in fp32 (sums of 1024 terms, each rounded to 2^-24 of what it holds, through two
    layers and their norms), 2e-2 under bf16 autocast, as the layers' other tests."""
    torch.manual_seed(N)
    spec = mfb.RelativeBias(32, "distance", 8.0)
    trunk = TransformerTrunk(128, 2, ["mha", "mha"], relative_bias=spec, mha_impl=impl)
    for block in trunk.blocks:
        torch.nn.init.normal_(block.ada_ln[-1].bias, std=0.3)
        torch.nn.init.normal_(block.attn.bias_table, std=2.0)
    x, cond, coords, grad = torch.randn(3, N, 128), torch.randn(3, 128), torch.randn(3, N, 3) * 3, torch.randn(3, N, 128)
    mask = _pad_masks(form, 3, N)
    there = ~mask
    pairs = there[:, :, None] & there[:, None]
    want_buckets = mfb.distance_buckets(coords, spec.edges)
    results = []
    for device, low in (("cpu", False), ("cuda", impl == "auto")):
        net = copy.deepcopy(trunk).to(device)
        given = []
        net.blocks[0].attn.register_forward_pre_hook(lambda _, args, kw: given.append(kw["buckets"]), with_kwargs=True)
        with torch.autocast("cuda", BF16, enabled=low):
            out = net(x.to(device), cond.to(device), pad_mask=mask.to(device), coords=coords.to(device))
        (out.float() * grad.to(device)).sum().backward()
        assert torch.equal(given[0].cpu()[pairs], want_buckets[pairs])
        results.append([out.detach().float().cpu()] + [b.attn.bias_table.grad.cpu() for b in net.blocks])
        assert device == "cpu" or {b.attn._last_core_used for b in net.blocks} == {"dense" if low else "torch"}
    for a, b in zip(*results):
        assert (a - b).abs().max() <= (2e-2 if impl == "auto" else 1e-3) * a.abs().max()


@pytest.mark.parametrize("form", ["front", "random"])
def test_a_model_with_padding_anywhere(form):
    """The same through a model, in fp32: two devices, one answer."""
    torch.manual_seed(1)
    model = EDMModel(d_model=64, n_heads=2, n_layers=2, attn_types=["mha", "mha"], relative_bias=mfb.RelativeBias(16, "distance", 6.0))
    for block in model.trunk.blocks:
        torch.nn.init.normal_(block.ada_ln[-1].bias, std=0.3)
        torch.nn.init.normal_(block.attn.bias_table, std=2.0)
    atoms, coords, sigma, mask = torch.randn(3, 21, 6), torch.randn(3, 21, 3) * 2, torch.rand(3) + 0.2, _pad_masks(form, 3, 21)
    want = model(atoms, coords, mask, sigma)
    got = copy.deepcopy(model).cuda()(atoms.cuda(), coords.cuda(), mask.cuda(), sigma.cuda())
    for a, b in zip(got, want):
        assert (a.cpu() - b)[~mask].abs().max() <= 1e-3 * b.abs().max()


@pytest.mark.parametrize("dtype", [BF16, torch.float16])
@pytest.mark.parametrize("bias", ["none", "offset", "pair"])
@pytest.mark.parametrize("backend", ["auto", "mma", "tcgen05"], indirect=True)
@pytest.mark.parametrize("B,H,K,M,N,D", [
    (2, 2, 2, 9, 29, 64),      # small entries
    (2, 4, 2, 1, 100, 64),     # few queries, one piece
    (2, 4, 2, 2, 2000, 128),   # up to 32 pieces
    (1, 2, 2, 1, 32768, 64),   # more
    (1, 2, 1, 300, 2500, 128), # tiles of 128 queries, keys in pieces
    (1, 2, 2, 300, 700, 64),   # the same in one piece
    (1, 2, 2, 70, 130, 32),
])  # fmt: skip
def test_what_is_no_number_stays_none(backend, B, H, K, M, N, D, bias, dtype):
    """A row that sees a logit that is not a number is none, whatever the sizes: a query of NaN, and a whole stretch of keys (with the others' rows as they
    are without it); its log-sum-exp is none either, so that the gradients show it."""
    g, q, k, v, grad = operands(M + N, B, H, K, M, N, D, dtype)
    table = buckets = None
    if bias != "none":
        table = torch.randn(16, H, generator=g, device="cuda")
        buckets = mfb.offset_buckets(16, 40, device="cuda") if bias == "offset" else torch.randint(0, 18, (B, M, N), generator=g, device="cuda", dtype=torch.uint8)

    def call(q, k):
        return mfb.dense_attention(q, k, v, bias=table, buckets=buckets)

    want = call(q, k)
    bad = q.clone()
    bad[-1, 1, M // 2] = NAN
    got = call(bad, k)
    assert got[-1, 1, M // 2].isnan().all()
    got[-1, 1, M // 2] = want[-1, 1, M // 2]
    assert torch.equal(got, want)
    for first, last in ((0, N), (N // 4, N - N // 4), (N - 1, N)):
        bad = k.clone()
        bad[-1, 0, first:last] = NAN
        got = call(q, bad)
        assert got[-1, : H // K].isnan().all()
        got[-1, : H // K] = want[-1, : H // K]
        assert torch.equal(got, want)
    leaf, keys = q.clone(), k.clone().requires_grad_()
    leaf[-1, 1, M // 2] = NAN
    leaf.requires_grad_()
    dq, dk = torch.autograd.grad(call(leaf, keys), [leaf, keys], grad)
    assert dq[-1, 1, M // 2].isnan().all() and dk[-1, 1 * K // H].isnan().all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("reach", [1, 5, 63, 64, 100, 190, 512])
@pytest.mark.parametrize("backend", ["tcgen05"], indirect=True)
def test_steps_at_either_end_of_the_map(backend, D, reach):
    """Steps of 64 keys whose offsets end or begin at the map's ends, where the sums along diagonals read its last entries."""
    for shift in (0, 1, reach % 64):
        M, N = 200, 200 + reach + shift
        g, q, k, v, grad = operands(reach + D, 1, 2, 2, M, N, D, BF16)
        table, buckets = torch.randn(16, 2, generator=g, device="cuda"), mfb.offset_buckets(16, reach, device="cuda")
        run_both(q, k, v, grad, bias=table, buckets=buckets)


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("backend", ["auto", "mma", "tcgen05"], indirect=True)
@pytest.mark.parametrize("M,N", [(40, 37), (70, 90), (200, 161), (300, 555)])
def test_pairs_of_one_row_for_all_queries(backend, M, N, D):
    """Buckets with a stride of zero over the queries, and rows that overlap, each ending with its storage: as a copy with rows of their own."""
    g, q, k, v, grad = operands(M + N, 2, 2, 2, M, N, D, BF16)
    table = torch.randn(16, 2, generator=g, device="cuda")
    store = torch.randint(0, 18, (N + 16 * (M - 1),), generator=g, device="cuda", dtype=torch.uint8)
    for buckets in (store[:N].expand(2, M, N), store[-N - 16 :][16:].expand(1, M, N), store.as_strided((1, M, N), (0, 16, 1)), store.as_strided((1, M, N), (0, 1, 1))):
        got = run_both(q, k, v, grad, bias=table, buckets=buckets)
        want = run_both(q, k, v, grad, bias=table, buckets=buckets.contiguous())
        if backend == "mma":
            assert all(torch.equal(got[n], want[n]) for n in want)


@pytest.mark.parametrize("backend", ["auto", "mma", "tcgen05"], indirect=True)
@pytest.mark.parametrize("one", [False, True])
@pytest.mark.parametrize("B,M,N", [(0, 50, 50), (2, 0, 50), (2, 50, 0), (2, 0, 0), (0, 0, 0)])
def test_empty_calls_by_pairs(backend, B, M, N, one):
    """Buckets of no pairs: zeros, forward and backward, as by offsets."""
    q, k, v = (torch.randn(B, 2, n, 64, device="cuda").to(BF16).requires_grad_() for n in (M, N, N))
    table = torch.randn(8, 2, device="cuda", requires_grad=True)
    buckets = torch.zeros(1 if one else B, M, N, device="cuda", dtype=torch.uint8)
    out = mfb.dense_attention(q, k, v, bias=table, buckets=buckets)
    assert out.shape == q.shape and not out.any()
    grads = torch.autograd.grad(out, [q, k, v, table], torch.ones_like(out))
    assert all(not g.any() and g.shape == t.shape for g, t in zip(grads, (q, k, v, table)))


@pytest.mark.parametrize("backend", ["auto", "mma", "tcgen05"], indirect=True)
@pytest.mark.parametrize("bias", ["none", "offset", "pair"])
@pytest.mark.parametrize("B,N", [(0, 50), (2, 0), (0, 0)])
def test_empty_packed_calls(backend, B, N, bias):
    qkv = torch.randn(B, N, 3 * 2 * 64, device="cuda").to(BF16).requires_grad_()
    table = None if bias == "none" else torch.randn(8, 2, device="cuda", requires_grad=True)
    buckets = {"none": None, "offset": mfb.offset_buckets(8, 10, device="cuda"), "pair": torch.zeros(1, N, N, device="cuda", dtype=torch.uint8)}[bias]
    out = mfb.dense_attention_packed(qkv, 2, bias=table, buckets=buckets)
    leaves = [qkv] if table is None else [qkv, table]
    grads = torch.autograd.grad(out, leaves, torch.ones_like(out))
    assert out.shape == (B, N, 128) and all(not g.any() and g.shape == t.shape for g, t in zip(grads, leaves))


def test_infinite_places_and_an_edge_at_zero():
    """An atom at infinity is no distance from itself: bucket 0, as on the CPU, whatever the edges."""
    x = torch.randn(2, 70, 3, generator=torch.Generator().manual_seed(0)) * 3
    x[0, 5, 1], x[1, 0, 0], x[1, 40, 2], x[1, 41, 2], x[0, 9] = NAN, math.inf, -math.inf, 3e38, math.inf
    x[0, 20] = x[0, 30]
    for edges in (torch.linspace(0.0, 12.0, 32, dtype=torch.float64), torch.zeros(3, dtype=torch.float64), torch.tensor([0.0, 0.0, 1.0, math.inf], dtype=torch.float64)):
        got = mfb.distance_buckets(x.cuda(), edges).cpu()
        assert torch.equal(got, mfb.distance_buckets(x, edges))
        assert got[1, 0, 0] == got[1, 40, 40] == got[0, 5, 5] == 0 and got[0, 0, 0] == got[0, 20, 30] == (edges == 0).sum()


@pytest.mark.parametrize("bias", ["none", "offset", "pair"])
@pytest.mark.parametrize("backend", ["auto", "mma", "tcgen05"], indirect=True)
@pytest.mark.parametrize("B,H,K,M,N,D", [(3, 2, 2, 29, 20, 64), (3, 2, 2, 20, 29, 32), (2, 4, 2, 90, 70, 64), (2, 2, 1, 300, 260, 64), (2, 2, 2, 300, 260, 128), (1, 2, 2, 130, 700, 32)])
def test_queries_that_see_nothing_may_hold_anything(backend, B, H, K, M, N, D, bias):
    """Causal entries with more queries than keys, or with keys hidden in front (a batch padded there): rows that see no key return zeros, and what they and
    their gradients hold reaches nobody else's."""
    g, q, k, v, grad = operands(M + N + D, B, H, K, M, N, D, BF16)
    key_mask = torch.rand(B, N, generator=g, device="cuda") < 0.9
    key_mask[:, : max(N // 3, N - M + M // 3)] = False
    table = buckets = None
    if bias != "none":
        table = torch.randn(16, H, generator=g, device="cuda")
        buckets = mfb.offset_buckets(16, 40, device="cuda") if bias == "offset" else torch.randint(0, 18, (B, M, N), generator=g, device="cuda", dtype=torch.uint8)
    i, j = torch.arange(M, device="cuda")[:, None], torch.arange(N, device="cuda")
    blind = ~((j - i <= N - M) & key_mask[:, None]).any(2)  # (B, M)
    assert blind.any()
    at = blind[:, None].expand(B, H, M)
    q[at], grad[at] = NAN, 0.0
    got = run_both(q, k, v, grad, key_mask=key_mask, causal=True, bias=table, buckets=buckets)
    assert not got["out"][at].any() and not got["dq"][at].any()
    q[at], grad[at] = math.inf, -math.inf
    leaves = [t.detach().requires_grad_() for t in (q, k, v)] + ([table.detach().requires_grad_()] if table is not None else [])
    out = mfb.dense_attention(*leaves[:3], key_mask=key_mask, causal=True, bias=leaves[-1] if table is not None else None, buckets=buckets)
    again = [out.detach(), *torch.autograd.grad(out, leaves, grad)]
    assert all(torch.equal(a, b) for a, b in zip(again, got.values()))


@pytest.mark.parametrize("N,row", [(1, 4), (5, 8), (29, 32), (30, 64), (129, 160), (131, 140)])
def test_bytes_behind_a_row(N, row):
    """Through the C interface, buckets as a part of a wider matrix (entries shorter than their rows): no byte but the pairs' own is written. In entries of whole
    rows the bytes behind are zeros or as they were, and what lies behind the entries stays."""
    x = torch.randn(2, N, 3, generator=torch.Generator().manual_seed(N)) * 3
    edges = torch.linspace(0.0, 8.0, 16, dtype=torch.float64)
    want, xc = mfb.distance_buckets(x, edges), x.cuda()
    for batch_stride in (N * row, N * row - 1, (N - 1) * row + N):
        store = torch.full((2 * N * row + 64,), 77, device="cuda", dtype=torch.uint8)
        _lib.launch(_lib.lib().mf_distance_buckets, xc.device, xc.data_ptr(), None, 2, N, edges.data_ptr(), edges.numel(), store.data_ptr(), batch_stride, row)
        out = store.as_strided((2, N, N), (batch_stride, row, 1))
        assert torch.equal(out.cpu(), want)
        out.fill_(77)
        if batch_stride == N * row:
            assert ((store == 77) | (store == 0))[: 2 * N * row].all() and (store[2 * N * row :] == 77).all()
        else:
            assert (store == 77).all()


@pytest.mark.parametrize("dtype", [torch.uint8, torch.float32])
def test_padding_masks_of_other_types(dtype):
    """The layer reads a padding mask of whole numbers, or of zeros and minus infinities, as it reads one of truth values: holes stay holes."""
    torch.manual_seed(0)
    layer = RegularAttention(128, 2, impl="cuda").cuda()
    x, mask = torch.randn(3, 40, 128, device="cuda"), _pad_masks("random", 3, 40).cuda()
    other = mask.to(dtype) if dtype == torch.uint8 else torch.zeros(3, 40, device="cuda").masked_fill(mask, -math.inf)
    with torch.no_grad(), torch.autocast("cuda", BF16):
        assert torch.equal(layer(x, key_padding_mask=other), layer(x, key_padding_mask=mask))


@pytest.mark.parametrize("bias", ["none", "offset", "pair"])
@pytest.mark.parametrize("B,H,K,M,N,D", [(1, 32, 1, 1, 4096, 128), (2, 71, 1, 1, 900, 64), (1, 34, 2, 3, 1500, 64), (2, 17, 1, 1, 1000, 32), (1, 20, 1, 5, 700, 128), (2, 64, 2, 1, 70, 64),
                                         (1, 24, 1, 40, 600, 64)])  # fmt: skip
def test_many_query_heads_on_a_key_head(B, H, K, M, N, D, bias):
    """More query heads to a key head than a tile has rows."""
    g, q, k, v, grad = operands(H + N, B, H, K, M, N, D, BF16)
    num_k, key_mask = counts(g, B, N), torch.rand(B, N, generator=g, device="cuda") < 0.8
    table = buckets = None
    if bias != "none":
        table = torch.randn(16, H, generator=g, device="cuda")
        table[3, H // 2] = -math.inf
        buckets = mfb.offset_buckets(16, 40, device="cuda") if bias == "offset" else torch.randint(0, 18, (B, M, N), generator=g, device="cuda", dtype=torch.uint8)
    run_both(q, k, v, grad, bias=table, buckets=buckets)
    run_both(q, k, v, grad, num_keys=num_k, key_mask=key_mask, causal=True, bias=table, buckets=buckets)


@pytest.mark.parametrize("scale", [1e-24, 3e-23, 1e-22, 2e-21, 1e-20, 1e-19, 1e-15, 1e15, 1e18, 5e18])
def test_distances_far_from_one(scale):
    """Squares that fp32 holds as subnormal numbers, as zeros or not at all, beside edges of their size, at distances that occur, and of another: as on the CPU."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 131, 3, generator=g) * scale
    x[1] = torch.randint(-4, 5, (131, 3), generator=g).float() * scale
    d = (x.double()[:, :, None] - x.double()[:, None]).norm(dim=-1).flatten()
    occur = d[torch.randint(0, len(d), (127,), generator=g)].sort().values
    for edges in (torch.linspace(0.0, 5 * scale, 32, dtype=torch.float64), occur, occur[:1], occur[-1:], occur * (1 + 1e-7), torch.linspace(0.0, 5.0, 32, dtype=torch.float64),
                  torch.tensor([0.0, scale, math.inf], dtype=torch.float64), torch.zeros(0, dtype=torch.float64)):  # fmt: skip
        assert torch.equal(mfb.distance_buckets(x.cuda(), edges).cpu(), mfb.distance_buckets(x, edges))


@pytest.mark.parametrize("axes", [1, 3])
@pytest.mark.parametrize("impl,biased", [("auto", False), ("cuda", False), ("auto", True)])
@pytest.mark.parametrize("N", [29, 60])
def test_padded_positions_that_are_no_numbers(N, impl, biased, axes):
    """Rotary positions of padding may hold anything: output and gradients as with zeros there."""
    torch.manual_seed(0)
    spec = mfb.RelativeBias(16, "offset", 6) if biased else None
    layer = RegularAttention(128, 2, impl=impl, relative_bias=spec, rotary=mfb.RotaryPositions(24, axes=axes)).cuda()
    x, mask = torch.randn(3, N, 128, device="cuda"), torch.arange(N, device="cuda") >= torch.tensor([N, N - 4, 3], device="cuda")[:, None]
    grad = torch.randn_like(x) * ~mask[..., None]
    more = {"buckets": spec.buckets(None, None, x.device)} if biased else {}
    places = torch.randn(3, N, *((axes,) if axes > 1 else ()), device="cuda")
    made = []
    for value in (0.0, NAN, math.inf):
        at = places.clone()
        at[mask] = value
        leaf = x.clone().requires_grad_()
        with torch.autocast("cuda", BF16):
            out = layer(leaf, key_padding_mask=mask, positions=at, **more)
        made.append([out[~mask], *torch.autograd.grad(out, [leaf, *layer.parameters()], grad.to(out.dtype))])
    for other in made[1:]:
        assert all(torch.equal(a, b) for a, b in zip(made[0], other))
