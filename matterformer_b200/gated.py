"""Gated feed-forward block: two projections, an activation of one times the other, and the projection back.

``gated_mlp(x, w_in, w_out, b_in, b_out)`` = ``(act(gate) * up) @ w_out.T + b_out`` with ``gate, up = (x @ w_in.T + b_in).chunk(2, -1)``,
the gated counterpart of the trunk's MLP (models/transformer.py:137-152 of the reference has the plain one; it has no operator of this
name).  Both projections, the activation and the product are one kernel, forward; backward, the gradient of the activation is
formed in the epilogue of the product that would otherwise store it.  All products run on this library's tcgen05 kernels.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
import torch.nn.functional as F

from . import _lib, simplicial
from .fused import watched
from .linear import bf16_copy

_ONCE = b"trying to differentiate twice a function that was marked with @once_differentiable"

_CODE = {torch.bfloat16: _lib.MF_DTYPE_BF16, torch.float16: _lib.MF_DTYPE_F16}
ACTIVATIONS = {"silu": _lib.MF_ACT_SILU, "gelu_tanh": _lib.MF_ACT_GELU_TANH}


def _ready(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """Contiguous and on a 16-byte boundary, as the kernels read it."""
    if t is None:
        return None
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _args(x, w_in, w_out, b_in, b_out, activation, grad_dtype):
    a = _lib.MfGatedMlpArgs()
    a.rows, a.dim, a.hidden, a.dim_out = x.shape[0], x.shape[1], w_out.shape[1], w_out.shape[0]
    a.dtype, a.activation = _CODE[x.dtype], ACTIVATIONS[activation]
    a.grad_dtype = _lib.MF_DTYPE_F32 if grad_dtype == torch.float32 else a.dtype
    a.x, a.w_in, a.w_out, a.b_in, a.b_out = _ptr(x), _ptr(w_in), _ptr(w_out), _ptr(b_in), _ptr(b_out)
    return a


def _raise_expired(device: torch.device) -> None:
    """After a call, where the caller has asked for it (see :func:`matterformer_b200.set_check_status`)."""
    if simplicial._CHECK_STATUS and not torch.cuda.is_current_stream_capturing():
        code = gated_mlp_status(device)
        if code != 0:
            raise RuntimeError(f"a device-side wait of the gated block's kernels expired (status {code}); the outputs of that call are undefined")


class _GatedMlp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_in, w_out, b_in, b_out, activation):
        ctx.shape, ctx.activation, ctx.grad_dtype = x.shape, activation, w_in.dtype
        x2 = _ready(x.reshape(-1, x.shape[-1]))
        params = [_ready(bf16_copy(p) if p is not None and p.dtype != x.dtype else p) for p in (w_in, w_out, b_in, b_out)]
        rows, hidden = x2.shape[0], w_out.shape[1]
        y = torch.empty((rows, w_out.shape[0]), device=x.device, dtype=x.dtype)
        act = torch.empty((rows, hidden), device=x.device, dtype=x.dtype)
        keep = any(ctx.needs_input_grad)
        pre = torch.empty(_lib.lib().mf_gated_mlp_pre_bytes(rows, hidden), device=x.device, dtype=torch.uint8) if keep else None
        a = _args(x2, *params, activation, ctx.grad_dtype)
        a.pre, a.act, a.y = _ptr(pre), _ptr(act), _ptr(y)
        L = _lib.lib()
        need = L.mf_gated_mlp_fwd_workspace_bytes(ctypes.byref(a))
        if need:
            ws = torch.empty(need, device=x.device, dtype=torch.uint8)
            a.workspace, a.workspace_bytes = ws.data_ptr(), need
        _lib.launch(L.mf_gated_mlp_fwd, x.device, ctypes.byref(a))
        _raise_expired(x.device)
        if keep:
            ctx.foreign = _lib.foreign_leaves(x, w_in, w_out, b_in, b_out)
            ctx.save_for_backward(x2, *params, pre, act)
        return y.view(*x.shape[:-1], w_out.shape[0])

    @staticmethod
    def backward(ctx, grad_y):
        _lib.refuse_foreign(ctx.foreign, "gated_mlp")
        with torch.no_grad():
            grads = _GatedMlp._gradients(ctx, grad_y)
        if torch.is_grad_enabled():  # create_graph: an error for who differentiates again, whichever operand the second gradient is of
            given = [g.requires_grad_() for g in grads if g is not None]
            made = torch._C._functions.DelayedError(_ONCE, len(given))(*given)
            made = iter((made,) if len(given) == 1 else made)
            grads = [None if g is None else next(made) for g in grads]
        return (*grads, None)

    @staticmethod
    def _gradients(ctx, grad_y):
        x, w_in, w_out, b_in, b_out, pre, act = ctx.saved_tensors
        grad_y = _ready(grad_y.reshape(-1, w_out.shape[0]).to(x.dtype))
        a = _args(x, w_in, w_out, b_in, b_out, ctx.activation, ctx.grad_dtype)
        wanted = [t if need else None for t, need in zip((x, w_in, w_out, b_in, b_out), ctx.needs_input_grad)]
        grads = [None if t is None else torch.empty(t.shape, device=x.device, dtype=x.dtype if i == 0 else ctx.grad_dtype)
                 for i, t in enumerate(wanted)]  # fmt: skip
        a.pre, a.act, a.grad_y = _ptr(pre), _ptr(act), _ptr(grad_y)
        a.grad_x, a.grad_w_in, a.grad_w_out, a.grad_b_in, a.grad_b_out = (_ptr(g) for g in grads)
        L = _lib.lib()
        need = L.mf_gated_mlp_bwd_workspace_bytes(ctypes.byref(a))
        ws = torch.empty(max(need, 16), device=x.device, dtype=torch.uint8)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
        _lib.launch(L.mf_gated_mlp_bwd, x.device, ctypes.byref(a))
        _raise_expired(x.device)
        if grads[0] is not None:
            grads[0] = grads[0].view(ctx.shape)
        return grads


def _plain(x, w_in, w_out, b_in, b_out, activation):
    """The block in torch operations, in ``x``'s type whatever autocast is for."""
    with torch.autocast(x.device.type, enabled=False):
        w_in, w_out, b_in, b_out = (None if p is None else p.to(x.dtype) for p in (w_in, w_out, b_in, b_out))
        gate, up = F.linear(x, w_in, b_in).chunk(2, dim=-1)
        return F.linear((F.silu(gate) if activation == "silu" else F.gelu(gate, approximate="tanh")) * up, w_out, b_out)


def gated_mlp_applies(x: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor) -> bool:
    """Whether the kernels take these operands: CUDA, 16-bit ``x``, parameters of its type (or fp32 beside bf16), widths that are
    multiples of 8."""
    return (x.is_cuda and x.dtype in _CODE and w_in.ndim == w_out.ndim == 2 and w_in.dtype == w_out.dtype
            and (w_in.dtype == x.dtype or (w_in.dtype == torch.float32 and x.dtype == torch.bfloat16))
            and all(n % 8 == 0 and 0 < n <= 2**28 for n in (w_in.shape[1], w_out.shape[1], w_out.shape[0])))  # fmt: skip


def _check(x, w_in, w_out, b_in, b_out, activation):
    if not x.is_cuda:
        raise RuntimeError("gated_mlp requires CUDA tensors")
    if activation not in ACTIVATIONS:
        raise ValueError(f"gated_mlp: activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    if x.dtype not in _CODE:
        raise RuntimeError(f"gated_mlp only supports float16/bfloat16 inputs, got {x.dtype}")
    params = [p for p in (w_in, w_out, b_in, b_out) if p is not None]
    if any(p.dtype != w_in.dtype for p in params) or not (w_in.dtype == x.dtype or (w_in.dtype, x.dtype) == (torch.float32, torch.bfloat16)):
        raise RuntimeError(f"gated_mlp: parameters must share the type of x, or be float32 beside bfloat16; got x {x.dtype}, "
                           f"parameters {[str(p.dtype) for p in params]}")  # fmt: skip
    if any(p.device != x.device for p in params):
        raise ValueError("gated_mlp: x and the parameters must be on one device")
    if x.ndim < 1 or w_in.ndim != 2 or w_out.ndim != 2 or w_in.shape != (2 * w_out.shape[1], x.shape[-1]):
        raise ValueError(f"gated_mlp: x (..., C), w_in (2 F, C) and w_out (O, F) expected, got {tuple(x.shape)}, {tuple(w_in.shape)}, "
                         f"{tuple(w_out.shape)}")  # fmt: skip
    if (b_in is not None and b_in.shape != w_in.shape[:1]) or (b_out is not None and b_out.shape != w_out.shape[:1]):
        raise ValueError("gated_mlp: b_in must have shape (2 F,) and b_out (O,)")
    if any(n < 8 or n % 8 or n > 2**28 for n in (x.shape[-1], *w_out.shape)):
        raise ValueError(f"gated_mlp: widths must be positive multiples of 8 up to 2^28, got C={x.shape[-1]}, F={w_out.shape[1]}, O={w_out.shape[0]}")


def gated_mlp(x: torch.Tensor, w_in: torch.Tensor, w_out: torch.Tensor, b_in: Optional[torch.Tensor] = None,
              b_out: Optional[torch.Tensor] = None, *, activation: str = "silu") -> torch.Tensor:  # fmt: skip
    """``x`` (..., C) bf16 or fp16; ``w_in`` (2 F, C) with the gate's rows first, ``w_out`` (O, F), biases (2 F,) and (O,) or None, of
    ``x``'s type, or fp32 beside a bf16 ``x`` (their bf16 copies compute, their gradients are fp32; see
    :func:`matterformer_b200.linear.bf16_copies`).  ``activation``: "silu" or "gelu_tanh".  Returns (..., O) in ``x``'s type.

    Sums are in fp32 in a fixed order.  The hidden values and the gradients of the pre-activations are rounded to ``x``'s type; hidden values
    that fp16 cannot hold (above 65504) are infinities there.  What the backward pass gets of the pre-activations has more bits than
    ``x``'s type, counted from the power of two in the largest of 16 neighbouring hidden channels of a token: 11 down to 2^-28 of that (bf16);
    13 where all are above 2^-7 of it, else 12 down to 2^-13 and one less for each halving beyond (fp16).  C, F and O are multiples of 8, at most 2^28.  The gradient is once differentiable.  What is traced
    or under a transform of ``torch.func`` is the same in plain operations, rounded after each."""
    native = None if simplicial._CHECK_STATUS else _lib.native()
    if native is not None and activation in ACTIVATIONS:  # operands that are ready as they are: one call into C++
        out = native.gated_mlp(x, w_in, w_out, b_in, b_out, ACTIVATIONS[activation])
        if out is not None:
            return out
    _check(x, w_in, w_out, b_in, b_out, activation)
    if watched(*(t for t in (x, w_in, w_out, b_in, b_out) if t is not None)):
        return _plain(x, w_in, w_out, b_in, b_out, activation)
    return _GatedMlp.apply(x, w_in, w_out, b_in, b_out, activation)


def gated_mlp_status(device=None) -> int:
    """0, or the code of a device-side wait that expired in one of the block's calls on the device since this was last asked; the outputs
    of that call are undefined.  Synchronises the current stream.  :func:`set_check_status` asks after every call."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    out = ctypes.c_int32(0)
    _lib.launch(_lib.lib().mf_gated_mlp_status, dev, ctypes.byref(out))
    return int(out.value)
