"""Rotary positions on queries and keys, in the layouts that attention layers have them.

The reference turns the heads of ``RotaryMultiheadAttention`` by 3-D positions before its attention core
(src/matterformer/models/regular_attention.py:208-271).  Here rotary positions are one operator for any table of frequencies, pairs of channels
half a rotation apart or next to each other, a part of the head, positions in a sequence or coordinates (pairs axis by axis, halves over all
axes; not compared with the order of the reference's pairs): :func:`rotary_embedding` on head-major
``q, k`` and :func:`rotary_packed` on the packed projection that :func:`matterformer_b200.sparse.local_window_attention_packed` takes.
Angles are formed in 64 bits, so that positions of millions keep theirs.
"""
from __future__ import annotations

import ctypes
import functools
import math
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib
from .fused import watched
from .simplicial import _DTYPE_CODE

MAX_PAIRS = 128


def rotary_frequencies(rotary_dim: int, *, axes: int = 1, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       original_length: Optional[float] = None, slow: float = 1.0, fast: float = 32.0) -> torch.Tensor:  # fmt: skip
    """Radians per unit of position for ``rotary_dim`` channels: ``(pairs,)`` or, for several axes, ``(axes, pairs)``, fp64 on the host, where
    the operators want it.  ``base ** (-p / pairs)``, for positions ``factor`` times as long as those a model knows scaled by

    * ``"linear"``: divided by ``factor`` (positions are interpolated);
    * ``"ntk"``: with a base ``factor ** (pairs / (pairs - 1))`` times as large: the last frequency is divided by ``factor``, the first stays;
    * ``"parts"``: frequencies that turn more than ``fast`` times within ``original_length`` stay, those that turn less than ``slow``
      times are divided by ``factor``, and between the two they go over linearly in the number of turns."""
    if axes < 1 or rotary_dim < 2 * axes or rotary_dim % (2 * axes):
        raise ValueError(f"rotary_dim must be a positive multiple of 2 * axes, got {rotary_dim} for {axes} axes")
    if not (base > 0.0 and math.isfinite(base)) or not (factor > 0.0 and math.isfinite(factor)):
        raise ValueError(f"base and factor must be positive, got {base} and {factor}")
    if scaling not in ("none", "linear", "ntk", "parts"):
        raise ValueError(f"scaling must be 'none', 'linear', 'ntk' or 'parts', got {scaling!r}")
    pairs = rotary_dim // (2 * axes)
    if scaling == "ntk" and pairs > 1:
        base = base * factor ** (pairs / (pairs - 1))
    theta = base ** (-torch.arange(pairs, dtype=torch.float64, device="cpu") / pairs)
    if scaling == "linear" or (scaling == "ntk" and pairs == 1):
        theta = theta / factor
    elif scaling == "parts":
        if original_length is None or not original_length > 0.0 or not fast > slow:
            raise ValueError("scaling 'parts' needs a positive original_length and fast > slow")
        kept = ((original_length * theta / (2.0 * math.pi) - slow) / (fast - slow)).clamp(0.0, 1.0)
        theta = kept * theta + (1.0 - kept) * theta / factor
    return theta if axes == 1 else theta.repeat(axes, 1)


@dataclass(frozen=True)
class RotaryPositions:
    """How an attention layer turns its queries and keys: the arguments of :func:`rotary_frequencies` and of :func:`rotary_embedding`."""

    rotary_dim: int
    axes: int = 1
    base: float = 10000.0
    layout: str = "half"
    amplitude: float = 1.0
    scaling: str = "none"
    factor: float = 1.0
    original_length: Optional[float] = None
    slow: float = 1.0
    fast: float = 32.0

    def __post_init__(self) -> None:
        if self.layout not in _lib.MF_ROTARY:
            raise ValueError(f"layout must be one of {sorted(_lib.MF_ROTARY)}, got {self.layout!r}")
        if not math.isfinite(self.amplitude):
            raise ValueError(f"amplitude must be finite, got {self.amplitude}")

    @functools.cached_property
    def frequencies(self) -> torch.Tensor:
        with torch.inference_mode(False):  # (kept: an ordinary tensor, whoever asks first)
            return rotary_frequencies(self.rotary_dim, axes=self.axes, base=self.base, scaling=self.scaling, factor=self.factor,
                                      original_length=self.original_length, slow=self.slow, fast=self.fast)  # fmt: skip


def rotate_torch(x: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, layout: str = "half", amplitude: float = 1.0) -> torch.Tensor:
    """:func:`rotary_embedding` of one (B, H, N, D) tensor in plain torch operations, on any device; angles in 64 bits."""
    if layout not in _lib.MF_ROTARY:
        raise ValueError(f"layout must be one of {sorted(_lib.MF_ROTARY)}, got {layout!r}")
    table = frequencies.to(positions.device)
    angle = positions.double()[..., None] * table if table.ndim == 1 else (positions.double()[..., None] * table).flatten(-2)
    if angle.ndim == 2:
        angle = angle[None]
    wide = torch.promote_types(x.dtype, torch.float32)
    cos, sin = (amplitude * f(angle[:, None]).to(wide) for f in (torch.cos, torch.sin))
    P = cos.shape[-1]
    a, b = (x[..., :P], x[..., P : 2 * P]) if layout == "half" else (x[..., 0 : 2 * P : 2], x[..., 1 : 2 * P : 2])
    a, b = a.to(wide), b.to(wide)
    turned = (a * cos - b * sin, a * sin + b * cos)
    turned = torch.cat(turned, dim=-1) if layout == "half" else torch.stack(turned, dim=-1).flatten(-2)
    return torch.cat([turned.to(x.dtype), x[..., 2 * P :]], dim=-1)


def rotate_packed_torch(qkv: torch.Tensor, heads: int, positions: torch.Tensor, frequencies: torch.Tensor, layout: str = "half",
                        amplitude: float = 1.0) -> torch.Tensor:  # fmt: skip
    """:func:`rotary_packed` in plain torch operations, on any device."""
    q, k, v = qkv.unflatten(-1, (3, heads, -1)).unbind(-3)  # (B, N, H, D) each
    q, k = (rotate_torch(t.transpose(1, 2), positions, frequencies, layout, amplitude).transpose(1, 2) for t in (q, k))
    return torch.stack([q, k, v], dim=-3).flatten(-3)


def _fill(tensor, x, out, heads, rotates, strides_in, strides_out):
    tensor.input, tensor.out, tensor.heads, tensor.rotates = x, out, heads, rotates
    tensor.in_batch, tensor.in_token, tensor.in_head = strides_in
    tensor.out_batch, tensor.out_token, tensor.out_head = strides_out


class _Rotary(torch.autograd.Function):
    """``heads`` 0: up to two head-major tensors; otherwise one packed projection with that many heads."""

    @staticmethod
    def forward(ctx, a, b, positions, table, heads, layout, amplitude, inverse):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions.clone() if positions.is_inference() else positions)
        ctx.call = (table.clone(), heads, layout, amplitude, inverse)  # (the caller's table may have changed by then)
        ctx.foreign = _lib.foreign_leaves(a, b)
        args = _lib.MfRotaryArgs()
        tensors = [t if t is None or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous() for t in (a, b)]
        x = next(t for t in tensors if t is not None)
        outs = [None if t is None else torch.empty_like(t) for t in tensors]
        # (overlapping inputs may have another order)
        outs = [o if o is None or o.stride(-1) == 1 else torch.empty(o.shape, dtype=o.dtype, device=o.device) for o in outs]
        if heads:
            args.batch, args.tokens = x.shape[:2]
            args.head_dim, args.tensors = x.shape[2] // (3 * heads), 3
            size, D = x.element_size(), args.head_dim
            for i in range(3):
                at = i * heads * D * size
                _fill(args.tensor[i], x.data_ptr() + at, outs[0].data_ptr() + at, heads, int(i < 2), (*x.stride()[:2], D), (*outs[0].stride()[:2], D))
        else:
            args.batch, args.tokens, args.head_dim = x.shape[0], x.shape[2], x.shape[3]
            for t, o in zip(tensors, outs):
                if t is not None:
                    s, z = t.stride(), o.stride()
                    _fill(args.tensor[args.tensors], t.data_ptr(), o.data_ptr(), t.shape[1], 1, (s[0], s[2], s[1]), (z[0], z[2], z[1]))
                    args.tensors += 1
        args.axes, args.pairs = (1, table.shape[0]) if table.ndim == 1 else table.shape
        args.dtype, args.layout, args.inverse, args.amplitude = _DTYPE_CODE[x.dtype], _lib.MF_ROTARY[layout], int(inverse), float(amplitude)
        args.position_type, args.positions = _lib.MF_POSITION[positions.dtype], positions.data_ptr()
        args.position_batch = positions.stride(0) if positions.ndim == (2 if table.ndim == 1 else 3) else 0
        args.frequencies = ctypes.cast(table.data_ptr(), ctypes.POINTER(ctypes.c_double))
        _lib.launch(_lib.lib().mf_rotary, x.device, ctypes.byref(args))
        return outs[0] if b is None else tuple(outs)

    @staticmethod
    def backward(ctx, *grads):
        _lib.refuse_foreign(ctx.foreign, "rotary_embedding")
        (positions,), (table, heads, layout, amplitude, inverse) = ctx.saved_tensors, ctx.call
        given = [g for g in grads if g is not None]  # (one of two outputs may be unused)
        out = [None] * 8
        if given:
            turned = _Rotary.apply(given[0], given[1] if len(given) > 1 else None, positions, table, heads, layout, amplitude, not inverse)
            turned = list(turned) if len(given) > 1 else [turned]
            for i, g in enumerate(grads):
                out[i] = turned.pop(0) if g is not None else None
        return tuple(out)


def _check(name, tensors, tokens, batch, heads, head_dim, positions, frequencies, layout, amplitude):
    x = tensors[0]
    if any(t.device.type != "cuda" for t in tensors):
        raise RuntimeError(f"{name} requires CUDA tensors")
    if x.dtype not in _DTYPE_CODE:
        raise RuntimeError(f"{name} only supports float16/bfloat16/float32 inputs, got {x.dtype}")
    if any(t.dtype != x.dtype or t.device != x.device for t in tensors):
        raise ValueError(f"{name}: tensors must share their type and device")
    if max(batch, tokens) >= 2**31 or heads * head_dim > 2**27:
        raise ValueError(f"{name}: fewer than 2^31 batch entries and tokens and at most 2^27 elements a token, got {batch}, {tokens} and {heads * head_dim}")
    if layout not in _lib.MF_ROTARY:
        raise ValueError(f"{name}: layout must be one of {sorted(_lib.MF_ROTARY)}, got {layout!r}")
    if not math.isfinite(amplitude):
        raise ValueError(f"{name}: amplitude must be finite, got {amplitude}")
    if not isinstance(frequencies, torch.Tensor) or frequencies.device.type != "cpu" or frequencies.ndim not in (1, 2) or frequencies.requires_grad:
        raise ValueError(f"{name}: frequencies must be a host tensor (pairs,) or (axes, pairs) without a gradient (see rotary_frequencies)")
    if not 1 <= frequencies.numel() <= MAX_PAIRS or 2 * frequencies.numel() > head_dim:
        raise ValueError(f"{name}: between 1 and min({MAX_PAIRS}, head_dim / 2) pairs, got {frequencies.numel()} for head_dim {head_dim}")
    axes = () if frequencies.ndim == 1 else (frequencies.shape[0],)
    if positions.dtype not in _lib.MF_POSITION:
        raise ValueError(f"{name}: positions must be int32, int64, float32 or float64, got {positions.dtype}")
    if positions.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name}: positions get no gradient; pass them detached")
    if positions.device != x.device or positions.shape not in ((tokens, *axes), (batch, tokens, *axes)):
        raise ValueError(f"{name}: positions of shape {(batch, tokens, *axes)} or {(tokens, *axes)} on {x.device} expected, got "
                         f"{tuple(positions.shape)} on {positions.device}")  # fmt: skip


def _ready(a, b, positions, frequencies, heads, layout, amplitude):
    """The whole call in C++ where that is built and the operands are ready as they are, else None."""
    native, code = _lib.native(), _lib.MF_ROTARY.get(layout)
    if native is None or code is None or not (isinstance(positions, torch.Tensor) and isinstance(frequencies, torch.Tensor)):
        return None
    return native.rotary(a, b, positions, frequencies, heads, code, amplitude)


def _apply(a, b, positions, frequencies, heads, layout, amplitude):
    if watched(*(t for t in (a, b, positions) if t is not None)):  # plain operations, which whatever watches can see
        if heads:
            return rotate_packed_torch(a, heads, positions, frequencies, layout, amplitude)
        turned = [rotate_torch(t, positions, frequencies, layout, amplitude) for t in (a, b) if t is not None]
        return turned[0] if b is None else tuple(turned)
    positions, table = positions.detach().contiguous(), frequencies.double().contiguous()
    return _Rotary.apply(a, b, positions, table, heads, layout, float(amplitude), False)


def rotary_embedding(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, frequencies: torch.Tensor, *,
                     layout: str = "half", amplitude: float = 1.0):  # fmt: skip
    """``q`` (B, H, N, D) and ``k`` (B, K, N, D) or None with the first ``2 * frequencies.numel()`` channels of every head turned by
    ``position * frequency`` and scaled by ``amplitude``; the channels behind them are copied.  Returns ``(q', k')``, k' None for None.

    ``layout``: "half" pairs channels p and p + P (P pairs in all), "interleaved" 2 p and 2 p + 1.  ``positions``: (N,) or (B, N) for frequencies
    (pairs,); (N, A) or (B, N, A) for frequencies (A, pairs), whose pairs follow each other axis by axis; integer or floating.  ``frequencies``: on the
    host (:func:`rotary_frequencies`).  Any strides with adjacent channels; results have the strides of dense inputs.  Differentiable
    in ``q`` and ``k``."""
    out = _ready(q, k, positions, frequencies, 0, layout, amplitude)
    if out is not None:
        return (out[0], None) if k is None else tuple(out)
    tensors = [t for t in (q, k) if t is not None]
    if any(t.ndim != 4 for t in tensors) or (k is not None and (k.shape[0], k.shape[2:]) != (q.shape[0], q.shape[2:])):
        raise ValueError(f"rotary_embedding: q (B, H, N, D) and k (B, K, N, D) expected, got {[tuple(t.shape) for t in tensors]}")
    _check("rotary_embedding", tensors, q.shape[2], q.shape[0], max(t.shape[1] for t in tensors), q.shape[3], positions, frequencies, layout, amplitude)
    out = _apply(q, k, positions, frequencies, 0, layout, amplitude)
    return (out, None) if k is None else out


def rotary_packed(qkv: torch.Tensor, heads: int, positions: torch.Tensor, frequencies: torch.Tensor, *, layout: str = "half",
                  amplitude: float = 1.0) -> torch.Tensor:  # fmt: skip
    """:func:`rotary_embedding` on the packed projection of an attention layer, ``qkv`` (B, N, 3*H*D): queries and keys turned, values copied."""
    out = _ready(qkv, None, positions, frequencies, int(heads), layout, amplitude) if heads >= 1 else None
    if out is not None:
        return out[0]
    if qkv.ndim != 3 or heads < 1 or qkv.shape[2] % (3 * heads) or qkv.shape[2] == 0:
        raise ValueError(f"rotary_packed: qkv (B, N, 3*H*D) with H = {heads} expected, got {tuple(qkv.shape)}")
    _check("rotary_packed", [qkv], qkv.shape[1], qkv.shape[0], heads, qkv.shape[2] // (3 * heads), positions, frequencies, layout, amplitude)
    return _apply(qkv, None, positions, frequencies, int(heads), layout, amplitude)
