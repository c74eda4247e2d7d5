"""Dense attention and distance buckets where inputs are unusual, as far as no GPU is needed (see test_dense_attention_edges_gpu.py)."""
import ctypes

import pytest
import torch
from test_dense_attention import BIAS, _args

import matterformer_b200 as mfb
from matterformer_b200 import _lib
from matterformer_b200.dense import dense_attention_torch
from matterformer_b200.trunk import RegularAttention


def test_buckets_of_no_pairs_have_no_address():
    L = _lib.lib()
    pairs = {**BIAS, "bucket_kind": _lib.MF_BUCKETS_PAIR, "buckets": None}
    for over in ({"batch": 0}, {"queries": 0}, {"queries": 0, "keys": 0}):
        assert L.mf_dense_attn_fwd(ctypes.byref(_args(**{**pairs, **over})), None) == _lib.MF_OK  # nothing to do
    for over in ({}, {"bucket_kind": _lib.MF_BUCKETS_OFFSET, "queries": 0}, {"bias": None, "queries": 0}):
        assert L.mf_dense_attn_fwd(ctypes.byref(_args(**{**pairs, **over})), None) == _lib.MF_ERR_INVALID_ARGUMENT
        assert "go together" in _lib.last_error()


def test_plain_form_under_autocast():
    """In fp32 whatever autocast is for, forward and backward, in the function and in a layer that has no kernel."""
    g = torch.Generator().manual_seed(0)
    q, k, v = (4 * torch.randn(2, 2, 40, 24, generator=g) for _ in range(3))
    table, buckets = torch.randn(8, 2, generator=g), mfb.offset_buckets(8, 10)
    for dtype in (torch.float32, torch.bfloat16):
        made = []
        for low in (False, True):
            leaves = [t.to(dtype).requires_grad_() for t in (q, k, v)] + [table.clone().requires_grad_()]
            with torch.autocast("cpu", torch.bfloat16, enabled=low):
                out = dense_attention_torch(*leaves[:3], bias=leaves[3], buckets=buckets, causal=True)
                plain = dense_attention_torch(*leaves[:3])
            assert out.dtype == dtype
            made.append([out, plain, *torch.autograd.grad(out.sum(), leaves)])
        assert all(torch.equal(a, b) for a, b in zip(*made))


def test_offsets_at_the_borders_of_buckets():
    """Beyond the first half of a side the bucket is the whole part of far * log(n / near) / log(reach / near), also where that is a whole number: compared by
    powers of whole numbers, without logarithms."""
    for num_buckets, reach in ((18, 128), (108, 64), (108, 125), (32, 128), (64, 512), (16, 64), (12, 27), (128, 1000)):
        side = num_buckets // 2
        near = side // 2
        far = side - near
        got = mfb.offset_buckets(num_buckets, reach).tolist()[: reach + 1][::-1]
        assert got[:near] == list(range(near))
        for n in range(near, reach + 1):
            k = got[n] - near
            assert n**far * near**k >= near**far * reach**k
            assert k == far - 1 or n**far * near ** (k + 1) < near**far * reach ** (k + 1)
    assert [mfb.offset_buckets(18, 128).tolist()[128 - n] for n in (7, 8, 15, 16, 31, 32, 63, 64)] == [4, 5, 5, 6, 6, 7, 7, 8]
