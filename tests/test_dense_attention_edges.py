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
