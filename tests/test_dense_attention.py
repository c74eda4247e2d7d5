"""Dense attention with a learned bias by buckets: the plain form, the buckets, what is refused, the layers that have it; no GPU."""
import ctypes
import math

import pytest
import torch
from torch import nn

import matterformer_b200 as mfb
from matterformer_b200 import _lib
from matterformer_b200.dense import dense_attention_torch
from matterformer_b200.trunk import AdaLNBlock, EDMModel, RegularAttention, TransformerTrunk

OK, OFF = 0x7F0000001000, 0x7F0000001002  # fake device addresses: validation never dereferences them


def _pair_by_pair(q, k, v, num_keys, num_queries, key_mask, causal, bias, buckets, scale):
    B, H, M, D = q.shape
    K, N = k.shape[1:3]
    out = torch.zeros_like(q)
    for b in range(B):
        nq, nk = (M if num_queries is None else int(num_queries[b])), (N if num_keys is None else int(num_keys[b]))
        for h in range(H):
            for i in range(nq):
                seen, logits = [], []
                for j in range(nk):
                    offset = j - i - (nk - nq)
                    if (causal and offset > 0) or (key_mask is not None and not key_mask[b, j]):
                        continue
                    z = scale * float(q[b, h, i] @ k[b, h * K // H, j])
                    if bias is not None:
                        L = len(buckets) // 2
                        which = int(buckets[max(-L, min(L, offset)) + L]) if buckets.ndim == 1 else int(buckets[b % buckets.shape[0], i, j])
                        value = float(bias[which, h]) if which < len(bias) else 0.0
                        if value < -1e30:
                            continue
                        z += value
                    seen.append(j)
                    logits.append(z)
                if seen:
                    top = max(logits)
                    w = [math.exp(z - top) for z in logits]
                    out[b, h, i] = sum(x / sum(w) * v[b, h * K // H, j] for x, j in zip(w, seen))
    return out


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("bias", ["none", "offset", "pair"])
@pytest.mark.parametrize("B,H,K,M,N", [(2, 4, 2, 5, 5), (3, 2, 1, 3, 7), (2, 2, 2, 6, 4), (1, 1, 1, 1, 1)])
def test_plain_form(B, H, K, M, N, bias, causal):
    g = torch.Generator().manual_seed(M * 10 + N)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    q, k, v = r(B, H, M, 8), r(B, K, N, 8), r(B, K, N, 8)
    num_k, num_q = torch.randint(0, N + 1, (B,), generator=g), torch.randint(0, M + 1, (B,), generator=g)
    mask = torch.rand(B, N, generator=g) < 0.8
    table = buckets = None
    if bias != "none":
        table = r(5, H)
        table[2, 0], table[1] = -math.inf, torch.finfo(torch.float32).min
        buckets = mfb.offset_buckets(4, 3) if bias == "offset" else torch.randint(0, 7, (B, M, N), generator=g, dtype=torch.uint8)
    for nk, nq, m in ((None, None, None), (num_k, num_q, None), (num_k, num_q, mask), (None, None, mask)):
        got = dense_attention_torch(q, k, v, nk, nq, key_mask=m, causal=causal, bias=table, buckets=buckets, scale=0.4)
        assert torch.allclose(got, _pair_by_pair(q, k, v, nk, nq, m, causal, table, buckets, 0.4), rtol=1e-12, atol=1e-12)
    hidden = ~mask
    bad_k, bad_v = k.clone(), v.clone()
    bad_k.transpose(1, 2)[hidden], bad_v.transpose(1, 2)[hidden] = math.nan, math.inf
    leaves = [t.clone().requires_grad_() for t in (q, bad_k, bad_v)]
    out = dense_attention_torch(*leaves, key_mask=mask, causal=causal, bias=table, buckets=buckets)
    assert torch.equal(out, dense_attention_torch(q, k, v, key_mask=mask, causal=causal, bias=table, buckets=buckets))
    assert all(torch.isfinite(t).all() for t in torch.autograd.grad(out.sum(), leaves))


def test_offset_buckets():
    got = mfb.offset_buckets(8, 10)
    assert got.dtype == torch.uint8 and got.tolist() == [3, 3, 3, 3, 3, 3, 2, 2, 2, 1, 0, 5, 6, 6, 6, 7, 7, 7, 7, 7, 7]
    one = mfb.offset_buckets(4, 6, bidirectional=False).tolist()
    assert one[:6] == [3, 3, 3, 2, 2, 1] and set(one[6:]) == {0}  # (the past backwards, then the present and what is never seen)
    for nb, reach in ((2, 1), (32, 128), (128, 1000), (6, 0)):
        b = mfb.offset_buckets(nb, reach).long()
        assert len(b) == 2 * reach + 1 and b.max() < nb
        past, later = b[: reach + 1].flip(0), b[reach + 1 :]
        assert (past.diff() >= 0).all() and (past < nb // 2).all() and (later.diff() >= 0).all() and (later >= nb // 2).all()
        assert torch.equal(later - nb // 2, past[1:])
    for nb, reach, both in ((7, 4, True), (0, 4, False), (130, 4, False), (8, -1, True), (1, 3, True)):
        with pytest.raises(ValueError, match="offset_buckets"):
            mfb.offset_buckets(nb, reach, bidirectional=both)


def test_distance_buckets():
    x = torch.tensor([[[0.0, 0, 0], [3, 4, 0], [0, 0, 1], [9, 9, 9]]])
    got = mfb.distance_buckets(x, [0.0, 1.0, 5.0, 5.0], torch.tensor([3]))
    assert got.dtype == torch.uint8 and got.tolist() == [[[1, 4, 2, 0], [4, 1, 4, 0], [2, 4, 1, 0], [0, 0, 0, 0]]]  # a distance at an edge is above it
    assert not mfb.distance_buckets(x, torch.zeros(0)).any()
    for edges, message in (([1.0, 0.5], "ascend"), ([-1.0], "ascend"), ([[1.0]], "vector"), ([float(i) for i in range(128)], "at most 127")):
        with pytest.raises(ValueError, match=message):
            mfb.distance_buckets(x, edges)
    with pytest.raises(ValueError, match="coords"):
        mfb.distance_buckets(x.double(), [1.0])
    with pytest.raises(ValueError, match="num_atoms"):
        mfb.distance_buckets(x, [1.0], torch.tensor([3, 3]))


@pytest.mark.parametrize("over", [{"num_buckets": 0}, {"num_buckets": 129}, {"kind": "angle"}, {"reach": 0.0}, {"reach": math.inf}, {"kind": "offset", "num_buckets": 5},
                                  {"kind": "offset", "reach": 2.5}])  # fmt: skip
def test_relative_bias_refusals(over):
    with pytest.raises(ValueError):
        mfb.RelativeBias(**over)


def _args(**over):
    rows = _lib.MfRows(4096, 512, 64)
    a = _lib.MfDenseAttnArgs(batch=2, heads=4, kv_heads=2, queries=100, keys=100, head_dim=64, dtype=_lib.MF_DTYPE_BF16, scale=0.125, q=OK, k=OK, v=OK, q_rows=rows, k_rows=rows,
                             v_rows=rows, out=OK, out_rows=rows, lse=OK, grad_out=OK, grad_out_rows=rows, dq=OK, dq_rows=rows)  # fmt: skip
    for name, value in over.items():
        setattr(a, name, value)
    return a


BIAS = {"bias": OK, "bias_dtype": _lib.MF_DTYPE_F32, "num_buckets": 8, "bucket_kind": 1, "reach": 4, "buckets": OK}


@pytest.mark.parametrize("over,message", [
    ({"dtype": _lib.MF_DTYPE_F32}, "bf16 or fp16"), ({"batch": -1}, "not negative"), ({"kv_heads": 3}, "multiple of kv_heads"), ({"heads": 0}, "multiple of kv_heads"),
    ({"head_dim": 48}, "32, 64 or 128"), ({"queries": 2**30}, "below 2"), ({"batch": 2**28}, "below 2"), ({"scale": math.inf}, "finite"), ({"scale": math.nan}, "finite"),
    ({"backend": 3}, "unknown backend"), ({"backend": -1}, "unknown backend"), ({"bias": OK}, "go together"), ({"buckets": OK}, "go together"),
    ({**BIAS, "bucket_kind": 0}, "go together"), ({**BIAS, "bucket_kind": 3}, "unknown bucket_kind"), ({**BIAS, "num_buckets": 129}, "between 1 and 128"),
    ({**BIAS, "num_buckets": 0}, "between 1 and 128"), ({**BIAS, "bias_dtype": 9}, "unknown bias_dtype"), ({**BIAS, "reach": -1}, "reach"),
    ({**BIAS, "bucket_kind": 2, "bucket_row": -1}, "not be negative"), ({"q": OFF}, "16-byte aligned"), ({"out": OFF}, "16-byte aligned"), ({"v": OFF}, "16-byte aligned"),
    ({"q_rows": _lib.MfRows(4096, 512, 60)}, "multiples of 8"), ({"k_rows": _lib.MfRows(4100, 512, 64)}, "multiples of 8"), ({"k": None}, "must not be NULL"),
    ({"out": None}, "must not be NULL"),
])  # fmt: skip
def test_arguments(over, message):
    L = _lib.lib()
    for fn in (L.mf_dense_attn_fwd, L.mf_dense_attn_bwd):
        assert fn(ctypes.byref(_args(**over)), None) == _lib.MF_ERR_INVALID_ARGUMENT
        assert message in _lib.last_error()
    assert L.mf_dense_attn_fwd_workspace_bytes(ctypes.byref(_args(**over))) == L.mf_dense_attn_bwd_workspace_bytes(ctypes.byref(_args(**over))) == 0


def test_more_arguments():
    L = _lib.lib()
    assert L.mf_dense_attn_fwd(None, None) == L.mf_dense_attn_bwd(None, None) == _lib.MF_ERR_INVALID_ARGUMENT
    assert L.mf_dense_attn_fwd_workspace_bytes(None) == L.mf_dense_attn_bwd_workspace_bytes(None) == 0
    assert L.mf_dense_attn_fwd(ctypes.byref(_args(batch=0, q=None)), None) == _lib.MF_OK  # nothing to do
    need = L.mf_dense_attn_bwd_workspace_bytes(ctypes.byref(_args()))
    assert need >= 2 * 4 * 100 * 4
    assert L.mf_dense_attn_bwd(ctypes.byref(_args()), None) == _lib.MF_ERR_WORKSPACE_TOO_SMALL
    assert L.mf_dense_attn_bwd(ctypes.byref(_args(workspace=OK, workspace_bytes=need - 1)), None) == _lib.MF_ERR_WORKSPACE_TOO_SMALL
    for over in ({"grad_out": None}, {"lse": None}, {"dk": OFF}, {"workspace": OFF}, {"dq_rows": _lib.MfRows(4096, 4, 64)}):
        assert L.mf_dense_attn_bwd(ctypes.byref(_args(**{"workspace": OK, "workspace_bytes": need, **over})), None) == _lib.MF_ERR_INVALID_ARGUMENT
    few = _args(queries=1, keys=100000)
    need = L.mf_dense_attn_fwd_workspace_bytes(ctypes.byref(few))
    assert need > 0 and L.mf_dense_attn_fwd(ctypes.byref(few), None) == _lib.MF_ERR_WORKSPACE_TOO_SMALL
    assert L.mf_dense_attn_status(None, None) == _lib.MF_ERR_INVALID_ARGUMENT
    status = ctypes.c_int32(0)
    for kind, limit, backend in ((5, 40000, 2), (-1, 40000, 2), (0, 9999, 2), (0, 2**31 + 1, 2), (0, 40000, 0)):
        assert L.mf_selftest_dense_attn_give_up(ctypes.byref(_args(backend=backend)), 0, kind, limit, ctypes.byref(status), None) == _lib.MF_ERR_INVALID_ARGUMENT
    edges = (ctypes.c_double * 200)(*range(200))
    ok = [OK, None, 2, 100, edges, 5, OK, 100 * 112, 112, None]
    for i, bad in ((2, -1), (3, 2**21), (5, 128), (5, -1), (0, None), (6, None), (8, 99), (7, 10000)):
        args = list(ok)
        args[i] = bad
        assert L.mf_distance_buckets(*args) == _lib.MF_ERR_INVALID_ARGUMENT, (i, bad)
    edges[1] = math.nan
    assert L.mf_distance_buckets(*ok) == _lib.MF_ERR_INVALID_ARGUMENT and "ascend" in _lib.last_error()
    assert ctypes.sizeof(_lib.MfDenseAttnArgs) == 10 * 4 + 3 * 8 + 3 * 24 + 3 * 8 + 8 + 8 + 4 * 4 + 3 * 8 + 8 + 24 + 8 + 8 + 24 + 3 * 8 + 3 * 24 + 3 * 8


def test_calls_that_are_refused():
    q = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="requires CUDA"):
        mfb.dense_attention(q, q, q)
    with pytest.raises(RuntimeError, match="requires CUDA"):
        mfb.dense_attention_packed(torch.zeros(1, 4, 192, dtype=torch.bfloat16), 1)
    with pytest.raises(ValueError, match="qkv"):
        mfb.dense_attention_packed(torch.zeros(1, 4, 100, dtype=torch.bfloat16), 1)
    with pytest.raises(ValueError, match="backend"):
        mfb.set_dense_backend("simt")


def _mask(B, N):
    mask = torch.arange(N) >= torch.tensor([N, N - 3, 2])[:B, None]
    return mask


def test_layer_with_a_table_of_zeros_is_the_plain_layer():
    torch.manual_seed(0)
    plain, biased = RegularAttention(64, 2), RegularAttention(64, 2, relative_bias=mfb.RelativeBias(8, "offset", 5))
    biased.attn.load_state_dict(plain.attn.state_dict())
    x, mask = torch.randn(3, 9, 64), _mask(3, 9)
    buckets = biased.relative_bias.buckets(None, None, x.device)
    want, got = plain(x, key_padding_mask=mask), biased(x, key_padding_mask=mask, buckets=buckets)
    assert torch.allclose(got[~mask], want[~mask], atol=1e-5)
    assert set(biased.state_dict()) - set(plain.state_dict()) == {"bias_table"}
    with torch.no_grad():
        biased.bias_table.normal_()
    out = biased(x, key_padding_mask=mask, buckets=buckets)
    assert not torch.allclose(out[~mask], want[~mask], atol=1e-3)
    out[~mask].square().sum().backward()
    assert biased.bias_table.grad.abs().max() > 0


def test_trunks_and_models():
    torch.manual_seed(0)
    coords, mask = torch.randn(3, 9, 3), _mask(3, 9)
    for kind in ("distance", "offset"):
        trunk = TransformerTrunk(64, 2, ["mha", "simplicial", "mha"], relative_bias=mfb.RelativeBias(8, kind, 4))
        for block in trunk.blocks:
            nn.init.normal_(block.ada_ln[-1].bias, std=0.3)
        more = {"coords": coords} if kind == "distance" else {}
        y = trunk(torch.randn(3, 9, 64), torch.randn(3, 64), pad_mask=mask, **more)
        y.square().sum().backward()
        assert [hasattr(b.attn, "bias_table") for b in trunk.blocks] == [True, False, True]
        assert all(b.attn.bias_table.grad.abs().max() > 0 for b in trunk.blocks if hasattr(b.attn, "bias_table"))
        assert "_offset_buckets" not in trunk.state_dict()
    model = EDMModel(d_model=64, n_heads=2, n_layers=2, relative_bias=mfb.RelativeBias(8))
    atoms, delta = model(torch.randn(3, 9, 6), coords, mask, torch.rand(3) + 0.1)
    assert torch.isfinite(atoms).all() and torch.isfinite(delta).all()
    with pytest.raises(ValueError, match="needs `coords`"):
        model.trunk(torch.randn(3, 9, 64), torch.randn(3, 64))
    with pytest.raises(ValueError, match="`coords` are for"):
        TransformerTrunk(64, 2, ["mha"])(torch.randn(3, 9, 64), torch.randn(3, 64), coords=coords)
    layer = RegularAttention(64, 2, relative_bias=mfb.RelativeBias(8))
    with pytest.raises(ValueError, match="needs `buckets`"):
        layer(torch.randn(3, 9, 64))
    with pytest.raises(ValueError, match="`buckets` are for"):
        RegularAttention(64, 2)(torch.randn(3, 9, 64), buckets=torch.zeros(9, 9, dtype=torch.uint8))
    with pytest.raises(ValueError, match="dropout"):
        RegularAttention(64, 2, dropout=0.1, relative_bias=mfb.RelativeBias(8))
    with pytest.raises(RuntimeError, match="dense attention kernels"):
        RegularAttention(64, 2, impl="cuda")(torch.randn(3, 9, 64))
    with pytest.raises(ValueError, match="Unsupported attention impl"):
        AdaLNBlock(64, 2, mha_impl="triton")


def test_distances_that_are_no_numbers_have_no_bucket():
    x = torch.zeros(1, 4, 3)
    x[0, 1, 0], x[0, 2, 1], x[0, 3, 2] = float("nan"), float("inf"), 1.5
    want = torch.tensor([[0, 0, 2, 1], [0, 0, 0, 0], [2, 0, 0, 2], [1, 0, 2, 0]], dtype=torch.uint8)
    assert torch.equal(mfb.distance_buckets(x, [1.0, 2.0])[0], want)
