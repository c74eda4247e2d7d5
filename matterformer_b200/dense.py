"""Dense attention with a learned bias by buckets.

The masked core of the reference's ``RotaryMultiheadAttention.forward`` (src/matterformer/models/regular_attention.py:208-271, additive mask into
``F.scaled_dot_product_attention``) over all keys of an entry, with the additive mask replaced by lengths, a key mask and an order, and by a
table of learned values: one for every bucket of pairs and head.  The reference has no operator of this kind; its geometry bias builders
(src/matterformer/models/transformer.py) write (B, H, N, N) tensors, which a table and one byte for each pair replace here.

:func:`dense_attention` and :func:`dense_attention_packed` are differentiable in the operands and in the table; the backward pass forms the
probabilities again.  :func:`offset_buckets` and :func:`distance_buckets` give the buckets: by place in a sequence, by distance of atoms.
"""
from __future__ import annotations

import ctypes
import functools
import math
import os
from dataclasses import dataclass
from typing import Optional, Sequence, Union

import torch

from . import _lib, simplicial
from .fused import watched

MAX_BUCKETS = 128
_CODE = {torch.bfloat16: _lib.MF_DTYPE_BF16, torch.float16: _lib.MF_DTYPE_F16}
_BIAS_CODE = {**_CODE, torch.float32: _lib.MF_DTYPE_F32}
_ONCE = b"trying to differentiate twice a function that was marked with @once_differentiable"
_BACKEND = os.environ.get("MF_DENSE_BACKEND", "auto")  # see set_dense_backend


def set_dense_backend(name: str) -> str:
    """Kernel family of dense attention: ``"auto"`` (by sizes), ``"mma"`` (warp-level tiles) or ``"tcgen05"`` (128-row tiles wherever they take
    the call).  Returns the previous setting."""
    global _BACKEND
    if name not in _lib.MF_DENSE_BACKEND:
        raise ValueError(f"unknown dense attention backend {name!r}")
    prev, _BACKEND = _BACKEND, name
    return prev


# ----------------------------------------------------------------------------------------------------------------------
# Buckets
# ----------------------------------------------------------------------------------------------------------------------
def offset_buckets(num_buckets: int, reach: int, *, bidirectional: bool = True, device=None) -> torch.Tensor:
    """Buckets of the offsets ``j - i`` = -reach .. reach of key and query, (2 * reach + 1,) uint8; offsets beyond fall into those of the ends.
    ``bidirectional``: the first half of the buckets for keys at or before the query, the second for later ones; otherwise all for
    the former, and later keys fall into the first.  Of a side's buckets the first half holds one offset each, the rest are spaced evenly
    over the logarithm up to ``reach``."""
    side = num_buckets // 2 if bidirectional else num_buckets
    if not 1 <= num_buckets <= MAX_BUCKETS or side < 1 or (bidirectional and num_buckets % 2):
        raise ValueError(f"offset_buckets: up to {MAX_BUCKETS} buckets, an even number for both directions, got {num_buckets}")
    if reach < 0:
        raise ValueError(f"offset_buckets: reach must not be negative, got {reach}")
    near = max(1, side // 2)
    far, (top, base) = side - near, (reach, near) if reach >= 2 * near else (2, 1)  # of the ratio that `far` buckets span
    spread = math.log(top / base)

    def beyond(n: int) -> int:
        """The whole part of far * log(n / near) / log(top / base); next to a whole number, which logarithms may miss, by powers of whole numbers."""
        x = math.log(n / near) / spread * far
        k = round(x)
        return int(x) if abs(x - k) > 1e-9 else k - (n**far * base**k < near**far * top**k)

    rank = [n if n < near else min(side - 1, near + beyond(n)) for n in range(reach + 1)]
    later = [side + r if bidirectional else 0 for r in rank[1:]]
    return torch.tensor(rank[::-1] + later, dtype=torch.uint8, device=device)


def _edges(edges: Union[torch.Tensor, Sequence[float]]) -> torch.Tensor:
    if isinstance(edges, torch.Tensor) and edges.device.type != "cpu":
        raise ValueError("distance_buckets: edges must be on the host")
    e = torch.as_tensor(edges, dtype=torch.float64).detach().contiguous()
    if e.ndim != 1 or e.numel() > MAX_BUCKETS - 1:
        raise ValueError(f"distance_buckets: edges must be a vector of at most {MAX_BUCKETS - 1} values, got shape {tuple(e.shape)}")
    if e.numel() and not (bool((e[1:] >= e[:-1]).all()) and 0.0 <= float(e[0])):
        raise ValueError("distance_buckets: edges must ascend from 0 on")
    return e


def _distance_buckets_torch(coords, edges, num_atoms):
    x = coords.detach().double()
    N = x.shape[1]
    d = x[:, :, None] - x[:, None]
    d2 = d[..., 0].square() + d[..., 1].square() + d[..., 2].square()
    out = torch.searchsorted(edges.square().to(x.device), d2.contiguous(), right=True)
    out = torch.where(d2.isnan(), 0, out)  # (a search takes what is not a number for the largest)
    if num_atoms is not None:
        real = torch.arange(N, device=x.device) < num_atoms.reshape(-1, 1)
        out = torch.where(real[:, :, None] & real[:, None], out, 0)
    return out.to(torch.uint8)


def distance_buckets(coords: torch.Tensor, edges: Union[torch.Tensor, Sequence[float]], num_atoms: Optional[torch.Tensor] = None) -> torch.Tensor:
    """(B, N, N) uint8: how many of the ascending ``edges`` (host values in fp64, at most 127, from 0 on) lie at or below the distance of two atoms of
    ``coords`` (B, N, 3) fp32, compared as squares in 64 bits.  0 where one of the two is padding (at or behind ``num_atoms`` (B))
    or where the distance is not a number.  On CUDA
    the rows start on 16-byte boundaries, as :func:`dense_attention` reads them fastest (the result is a view of a wider tensor).  No gradient."""
    native = _lib.native()
    if native is not None and isinstance(edges, torch.Tensor):
        out = native.distance_buckets(coords, edges, num_atoms)
        if out is not None:
            return out
    if coords.ndim != 3 or coords.shape[-1] != 3 or coords.dtype != torch.float32:
        raise ValueError(f"distance_buckets: coords (B, N, 3) float32 expected, got {tuple(coords.shape)} {coords.dtype}")
    B, N, _ = coords.shape
    e = _edges(edges)
    num = _counts("distance_buckets", "num_atoms", num_atoms, B, coords.device)
    if coords.device.type != "cuda" or watched(coords):
        return _distance_buckets_torch(coords, e, num)
    x = coords.detach().contiguous()
    row = -(-N // 16) * 16
    out = torch.empty((B, N, row), device=x.device, dtype=torch.uint8)
    _lib.launch(_lib.lib().mf_distance_buckets, x.device, x.data_ptr(), _ptr(num), B, N, e.data_ptr(), e.numel(), out.data_ptr(), N * row, row)
    return out[:, :, :N]


@dataclass(frozen=True)
class RelativeBias:
    """How an attention layer biases its logits: a learned table of ``num_buckets`` rows, one column for each head, that starts from zeros.  ``kind``: "distance" (of
    coordinates, in even steps up to ``reach``, beyond which all fall into the last bucket) or "offset" (of places in the sequence, :func:`offset_buckets` in
    both directions)."""

    num_buckets: int = 32
    kind: str = "distance"
    reach: float = 12.0

    def __post_init__(self) -> None:
        if self.kind not in ("distance", "offset"):
            raise ValueError(f"kind must be 'distance' or 'offset', got {self.kind!r}")
        if not 1 <= self.num_buckets <= MAX_BUCKETS or (self.kind == "offset" and self.num_buckets % 2):
            raise ValueError(f"up to {MAX_BUCKETS} buckets, an even number of them by offset, got {self.num_buckets}")
        if not (math.isfinite(self.reach) and self.reach > 0) or (self.kind == "offset" and self.reach != int(self.reach)):
            raise ValueError(f"reach must be positive, a whole number for buckets by offset, got {self.reach}")

    @functools.cached_property
    def edges(self) -> torch.Tensor:
        with torch.inference_mode(False):  # (kept: an ordinary tensor, whoever asks first)
            return torch.linspace(0.0, float(self.reach), self.num_buckets, dtype=torch.float64, device="cpu")[1:].contiguous()

    def buckets(self, positions: Optional[torch.Tensor], num_tokens: Optional[torch.Tensor], device) -> torch.Tensor:
        """As :func:`dense_attention` takes them; ``positions`` (B, N, 3) for distances.  ``num_tokens``: (B,) counts of real tokens, of entries
        whose padding is at the end; ``None`` for padding anywhere."""
        if self.kind == "offset":
            return offset_buckets(self.num_buckets, int(self.reach), device=device)
        return distance_buckets(positions.detach().float(), self.edges, num_tokens)


# ----------------------------------------------------------------------------------------------------------------------
# Attention
# ----------------------------------------------------------------------------------------------------------------------
def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _counts(name, what, num, batch, device):
    if num is None:
        return None
    if num.numel() != batch or num.dtype not in (torch.int32, torch.int64) or num.device != device:
        raise ValueError(f"{name}: {what} must hold one int32 or int64 count for each of {batch} entries on {device}, got shape {tuple(num.shape)} "
                         f"{num.dtype} on {num.device}")  # fmt: skip
    return num.detach().reshape(-1).to(torch.int32).contiguous()


def _ready(t: torch.Tensor) -> torch.Tensor:
    """Adjacent channels, rows on 16-byte boundaries."""
    fits = t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s % 8 == 0 for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1)
    return t if fits else t.contiguous() if not t.is_contiguous() else t.clone()


def _rows(t: torch.Tensor) -> "_lib.MfRows":
    b, h, n = (s if size > 1 else 0 for s, size in zip(t.stride()[:3], t.shape[:3]))
    return _lib.MfRows(b, h, n)


def _like(t: torch.Tensor) -> torch.Tensor:
    """A dense (B, H, N, D) tensor in the order of tokens and heads of ``t``."""
    B, H, N, D = t.shape
    if H > 1 and N > 1 and t.stride(1) < t.stride(2):
        return torch.empty((B, N, H, D), device=t.device, dtype=t.dtype).transpose(1, 2)
    return torch.empty((B, H, N, D), device=t.device, dtype=t.dtype)


def _split(qkv: torch.Tensor, heads: int):
    B, N, W = qkv.shape
    return qkv.view(B, N, 3, heads, W // (3 * heads)).permute(2, 0, 3, 1, 4).unbind(0)


def _args(q, k, v, num_queries, num_keys, key_mask, bias, buckets, causal, scale):
    a = _lib.MfDenseAttnArgs()
    a.batch, a.heads, a.queries, a.head_dim = q.shape
    a.kv_heads, a.keys = k.shape[1:3]
    a.dtype, a.causal, a.scale, a.backend = _CODE[q.dtype], int(causal), float(scale), _lib.MF_DENSE_BACKEND[_BACKEND]
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.q_rows, a.k_rows, a.v_rows = _rows(q), _rows(k), _rows(v)
    a.num_queries, a.num_keys = _ptr(num_queries), _ptr(num_keys)
    if key_mask is not None:
        a.key_mask, a.key_mask_batch = key_mask.data_ptr(), key_mask.stride(0)
    if bias is not None:
        a.bias, a.bias_dtype, a.num_buckets, a.buckets = bias.data_ptr(), _BIAS_CODE[bias.dtype], bias.shape[0], buckets.data_ptr()
        if buckets.ndim == 1:
            a.bucket_kind, a.reach = _lib.MF_BUCKETS_OFFSET, buckets.shape[0] // 2
        else:
            a.bucket_kind = _lib.MF_BUCKETS_PAIR
            a.bucket_batch, a.bucket_row = buckets.stride(0) if buckets.shape[0] > 1 else 0, buckets.stride(1)
    return a


def _workspace(a, need, device):
    if need:
        ws = torch.empty(need, device=device, dtype=torch.uint8)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
        return ws
    return None


class _DenseAttention(torch.autograd.Function):
    """``heads`` 0: head-major q, k, v; otherwise the packed projection with that many heads in the place of q."""

    @staticmethod
    def forward(ctx, q, k, v, bias, buckets, num_queries, num_keys, key_mask, heads, causal, scale):
        ctx.foreign = _lib.foreign_leaves(q, k, v, bias)
        ctx.call = (heads, causal, scale)
        if heads:
            packed = q.contiguous()
            given = [packed if packed.data_ptr() % 16 == 0 else packed.clone()]
            q, k, v = _split(given[0], heads)
        else:
            given = q, k, v = [_ready(t) for t in (q, k, v)]
        table = None if bias is None else bias.contiguous()
        a = _args(q, k, v, num_queries, num_keys, key_mask, table, buckets, causal, scale)
        out = _like(q)
        a.out, a.out_rows = out.data_ptr(), _rows(out)
        keep = any(ctx.needs_input_grad)
        lse = torch.empty(q.shape[:3], device=q.device, dtype=torch.float32) if keep else None
        a.lse = _ptr(lse)
        L = _lib.lib()
        ws = _workspace(a, L.mf_dense_attn_fwd_workspace_bytes(ctypes.byref(a)), q.device)  # noqa: F841 (until the launch)
        _lib.launch(L.mf_dense_attn_fwd, q.device, ctypes.byref(a))
        _raise_expired(q.device)
        out = out.transpose(1, 2).flatten(2) if heads else out
        if keep:
            aux = [t.clone() if t is not None and t.is_inference() else t for t in (buckets, num_queries, num_keys, key_mask)]
            ctx.save_for_backward(*given, table, out, lse, *aux)
        return out

    @staticmethod
    def backward(ctx, grad_out):
        _lib.refuse_foreign(ctx.foreign, "dense_attention")
        with torch.no_grad():
            grads = _DenseAttention._gradients(ctx, grad_out)
        if torch.is_grad_enabled():  # create_graph: an error for who differentiates again
            given = [g.requires_grad_() for g in grads if g is not None]
            made = torch._C._functions.DelayedError(_ONCE, len(given))(*given)
            made = iter((made,) if len(given) == 1 else made)
            grads = [None if g is None else next(made) for g in grads]
        return (*grads, *[None] * 7)

    @staticmethod
    def _gradients(ctx, grad_out):
        heads, causal, scale = ctx.call
        *given, table, out, lse, buckets, num_queries, num_keys, key_mask = ctx.saved_tensors
        grad_out = grad_out.to(out.dtype)
        if heads:
            q, k, v = _split(given[0], heads)
            out, grad_out = (t.unflatten(-1, (heads, q.shape[-1])).transpose(1, 2) for t in (out, grad_out))
            made = torch.empty_like(given[0])
            dq, dk, dv = _split(made, heads)
        else:
            q, k, v = given
            dq, dk, dv = (_like(t) if need else None for t, need in zip(given, ctx.needs_input_grad))
        grad_out = _ready(grad_out)
        dbias = torch.empty_like(table) if ctx.needs_input_grad[3] else None
        a = _args(q, k, v, num_queries, num_keys, key_mask, table, buckets, causal, scale)
        a.out, a.out_rows, a.lse = out.data_ptr(), _rows(out), lse.data_ptr()
        a.grad_out, a.grad_out_rows = grad_out.data_ptr(), _rows(grad_out)
        for name, t in (("dq", dq), ("dk", dk), ("dv", dv)):
            if t is not None:
                setattr(a, name, t.data_ptr())
                setattr(a, name + "_rows", _rows(t))
        a.dbias = _ptr(dbias)
        L = _lib.lib()
        ws = _workspace(a, L.mf_dense_attn_bwd_workspace_bytes(ctypes.byref(a)), q.device)  # noqa: F841
        _lib.launch(L.mf_dense_attn_bwd, q.device, ctypes.byref(a))
        _raise_expired(q.device)
        return [made if ctx.needs_input_grad[0] else None, None, None, dbias] if heads else [dq, dk, dv, dbias]


def dense_attention_status(device=None) -> int:
    """0, or the code of a device-side wait that expired in one of the dense attention calls on the device since this was last asked; the outputs
    of that call are undefined.  Synchronises the current stream.  :func:`set_check_status` asks after every call."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    out = ctypes.c_int32(0)
    _lib.launch(_lib.lib().mf_dense_attn_status, dev, ctypes.byref(out))
    return int(out.value)


def _raise_expired(device: torch.device) -> None:
    """After a call, where the caller has asked for it (see :func:`matterformer_b200.set_check_status`)."""
    if simplicial._CHECK_STATUS and not torch.cuda.is_current_stream_capturing():
        code = dense_attention_status(device)
        if code != 0:
            raise RuntimeError(f"a device-side wait of the dense attention kernels expired (status {code}); the outputs of that call are undefined")


def _lengths(num, most, device):
    return torch.full((1, 1, 1), most, device=device) if num is None else num.long().clamp(0, int(most)).reshape(-1, 1, 1)


def dense_attention_torch(q, k, v, num_keys=None, num_queries=None, *, key_mask=None, causal=False, bias=None, buckets=None, scale=None) -> torch.Tensor:
    """:func:`dense_attention` in plain torch operations, on any device and in any floating type (16-bit operands in fp32), whatever autocast is for."""
    with torch.autocast(q.device.type, enabled=False):
        return _plain(q, k, v, num_keys, num_queries, key_mask, causal, bias, buckets, scale)


def _plain(q, k, v, num_keys, num_queries, key_mask, causal, bias, buckets, scale):
    B, H, M, D = q.shape
    K, N = k.shape[1:3]
    wide = torch.promote_types(q.dtype, torch.float32)
    i, j = torch.arange(M, device=q.device)[:, None], torch.arange(N, device=q.device)
    nq, nk = _lengths(num_queries, M, q.device), _lengths(num_keys, N, q.device)
    offset = j - i - (nk - nq)  # (1 or B, M, N)
    see = (i < nq) & (j < nk)
    if causal:
        see = see & (offset <= 0)
    if key_mask is not None:
        see = see & key_mask[:, None, :]
    see = see.expand(B, M, N)
    # what no query sees, and queries that see nothing, may hold anything: their numbers do not enter
    shown, awake = see.any(1)[:, None, :, None], see.any(2)[:, None, :, None]
    qw = torch.where(awake, q.to(wide), 0.0)
    kw, vw = (torch.where(shown, t.to(wide), 0.0).repeat_interleave(int(H) // int(K), dim=1) for t in (k, v))
    logits = (qw @ kw.transpose(-1, -2)) * (D**-0.5 if scale is None else scale)
    see = see[:, None]
    if bias is not None:
        if buckets.ndim == 1:
            L = int(buckets.shape[0]) // 2
            which = buckets[offset.clamp(-L, L) + L].long()
        else:
            which = buckets.long()
        table = torch.cat([bias.to(wide), bias.new_zeros((256 - bias.shape[0], H), dtype=wide)])
        value = table[which].permute(0, 3, 1, 2)
        see = see & ~(value < -1e30)
        logits = logits + torch.where(see, value, 0.0)
    logits = torch.where(see, logits, torch.finfo(wide).min)
    p = torch.where(see, torch.softmax(logits, dim=-1), 0.0)
    return (p @ vw).to(q.dtype)


def _check(name, q, k, v, bias, buckets, key_mask, scale):
    if q.device.type != "cuda":
        raise RuntimeError(f"{name} requires CUDA tensors")
    if q.dtype not in _CODE:
        raise RuntimeError(f"{name} only supports float16/bfloat16 inputs, got {q.dtype}")
    if any(t.dtype != q.dtype or t.device != q.device for t in (k, v)):
        raise ValueError(f"{name}: q, k and v must share their type and device")
    if q.ndim != 4 or k.ndim != 4 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3] or k.shape[1] < 1 or q.shape[1] % k.shape[1] \
            or q.shape[1] < 1:  # fmt: skip
        raise ValueError(f"{name}: q (B, H, M, D), k and v (B, K, N, D) with H a multiple of K expected, got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    B, H, M, D = q.shape
    N = k.shape[2]
    if D not in (32, 64, 128):
        raise ValueError(f"{name}: head_dim must be 32, 64 or 128, got {D}")
    if not math.isfinite(scale):
        raise ValueError(f"{name}: scale must be finite, got {scale}")
    if (bias is None) != (buckets is None):
        raise ValueError(f"{name}: bias and buckets go together")
    if bias is not None:
        if bias.ndim != 2 or bias.shape[1] != H or not 1 <= bias.shape[0] <= MAX_BUCKETS or bias.dtype not in _BIAS_CODE or bias.device != q.device:
            raise ValueError(f"{name}: bias (buckets, {H}) with up to {MAX_BUCKETS} rows, float16, bfloat16 or float32 on {q.device} expected, got "
                             f"{tuple(bias.shape)} {bias.dtype} on {bias.device}")  # fmt: skip
        pairs = buckets.ndim in (2, 3) and buckets.shape[-2:] == (M, N) and (buckets.ndim == 2 or buckets.shape[0] in (1, B))
        if buckets.dtype != torch.uint8 or buckets.device != q.device or not (pairs or (buckets.ndim == 1 and buckets.shape[0] % 2 == 1)):
            raise ValueError(f"{name}: buckets uint8 of an odd number of offsets or of pairs (1 or {B}, {M}, {N}) on {q.device} expected, got "
                             f"{tuple(buckets.shape)} {buckets.dtype} on {buckets.device}")  # fmt: skip
    if key_mask is not None and (key_mask.shape != (B, N) or key_mask.dtype != torch.bool or key_mask.device != q.device):
        raise ValueError(f"{name}: key_mask ({B}, {N}) bool on {q.device} expected, got {tuple(key_mask.shape)} {key_mask.dtype} on {key_mask.device}")


def _aux(buckets, key_mask):
    if buckets is not None:
        buckets = buckets[None] if buckets.ndim == 2 else buckets
        if buckets.stride(-1) != 1 and buckets.shape[-1] > 1:
            buckets = buckets.contiguous()
    return buckets, None if key_mask is None else key_mask.contiguous()


def dense_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, num_keys: Optional[torch.Tensor] = None, num_queries: Optional[torch.Tensor] = None, *,
                    key_mask: Optional[torch.Tensor] = None, causal: bool = False, bias: Optional[torch.Tensor] = None,
                    buckets: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:  # fmt: skip
    """``q`` (B, H, M, D), ``k`` and ``v`` (B, K, N, D) bf16 or fp16, H a multiple of K (query head h reads key head h * K // H), D 32, 64 or 128, any
    strides with adjacent channels (expanded dimensions keep to the warp-level kernels; shared key heads are fastest as K heads).  Returns (B, H, M, D) with the tokens and heads in memory as ``q`` has them.

    ``num_keys``, ``num_queries``: (B,) counts of real keys and queries, which come first; what lies behind them may hold anything and returns
    zeros, as does a query that sees no key.  By counts, key mask and order: such a query, its gradient and keys that are hidden from all may hold anything; what the
    order hides from some queries, or the table hides, takes part in products and has to be numbers.  A query with a logit that is not a number returns none.  ``key_mask``: (B, N) bool, False hides a key.
    ``causal``: the last real query stands at the last real key, and no query sees later keys than its place.  ``bias``: a table (buckets, H) of up to 128 rows, fp32 or 16 bits, added to the logits
    ``scale * q . k`` (scale: D ** -0.5 by default) by the bucket of the pair; ``buckets``: uint8, either (2 L + 1,) for the offsets -L .. L between the place of the key
    and that of the query (:func:`offset_buckets`), which hold their ends for all beyond, or (B or 1, M, N) for every pair (:func:`distance_buckets`).  A
    bucket beyond the table has no bias; a value of minus infinity or below -1e30 hides its pairs.

    Softmax and sums are in fp32 in a fixed order; probabilities and the gradients of the logits are rounded to the operands' type before
    the products that contract them.  Once differentiable in q, k, v and the table.  What is traced or under a transform of
    ``torch.func`` is the same in plain operations."""
    native = None if simplicial._CHECK_STATUS else _lib.native()
    if native is not None:  # operands that are ready as they are: one call into C++
        out = native.dense_attention(q, k, v, bias, buckets, num_queries, num_keys, key_mask, 0, bool(causal), scale, _lib.MF_DENSE_BACKEND[_BACKEND])
        if out is not None:
            return out
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    _check("dense_attention", q, k, v, bias, buckets, key_mask, scale)
    num_keys = _counts("dense_attention", "num_keys", num_keys, q.shape[0], q.device)
    num_queries = _counts("dense_attention", "num_queries", num_queries, q.shape[0], q.device)
    buckets, key_mask = _aux(buckets, key_mask)
    if watched(*(t for t in (q, k, v, bias) if t is not None)):
        return dense_attention_torch(q, k, v, num_keys, num_queries, key_mask=key_mask, causal=causal, bias=bias, buckets=buckets, scale=scale)
    return _DenseAttention.apply(q, k, v, bias, buckets, num_queries, num_keys, key_mask, 0, bool(causal), scale)


def dense_attention_packed(qkv: torch.Tensor, heads: int, num_tokens: Optional[torch.Tensor] = None, *, key_mask: Optional[torch.Tensor] = None,
                           causal: bool = False, bias: Optional[torch.Tensor] = None, buckets: Optional[torch.Tensor] = None,
                           scale: Optional[float] = None) -> torch.Tensor:  # fmt: skip
    """:func:`dense_attention` of tokens on themselves on the packed projection of an attention layer: ``qkv`` (B, N, 3*H*D), result (B, N, H*D) as the output
    projection takes it, the gradient in ``qkv``'s shape."""
    native = None if simplicial._CHECK_STATUS else _lib.native()
    if native is not None and heads >= 1:
        out = native.dense_attention(qkv, None, None, bias, buckets, num_tokens, num_tokens, key_mask, int(heads), bool(causal), scale, _lib.MF_DENSE_BACKEND[_BACKEND])
        if out is not None:
            return out
    if qkv.ndim != 3 or heads < 1 or qkv.shape[2] % (3 * heads) or qkv.shape[2] == 0:
        raise ValueError(f"dense_attention_packed: qkv (B, N, 3*H*D) with H = {heads} expected, got {tuple(qkv.shape)}")
    q, k, v = _split(qkv.detach() if qkv.is_contiguous() else qkv.detach().contiguous(), heads)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    _check("dense_attention_packed", q, k, v, bias, buckets, key_mask, scale)
    num = _counts("dense_attention_packed", "num_tokens", num_tokens, qkv.shape[0], qkv.device)
    buckets, key_mask = _aux(buckets, key_mask)
    if watched(*(t for t in (qkv, bias) if t is not None)):
        q, k, v = qkv.unflatten(-1, (3, heads, -1)).permute(2, 0, 3, 1, 4).unbind(0)
        out = dense_attention_torch(q, k, v, num, num, key_mask=key_mask, causal=causal, bias=bias, buckets=buckets, scale=scale)
        return out.transpose(1, 2).flatten(2)
    return _DenseAttention.apply(qkv, None, None, bias, buckets, num, num, key_mask, int(heads), bool(causal), scale)
