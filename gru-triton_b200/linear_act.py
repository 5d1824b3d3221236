"""Matrix product with bias, activation and residual in its epilogue.

    y = act(x @ W^T + bias) + residual

The product that makes the gates of a recurrence, that widens a feed-forward layer, or that takes a layer's
output back into the stream of a model, without a second pass over its result.  ``tc.linear`` is its neighbour for
quantised weights: float32 alone, no activation or residual.

Element types float32, bfloat16 and float16, one for all tensors of a call; sums are float32.  float32 operands run as
two row-scaled fp16 planes in three tensor-core products (22 significant bits, as ``tc.linear``'s).  What the backward
needs of the activation is its slope, kept by the forward in float32 or, for the 16-bit types, in 16 bits: to 2^-16, and to 2^-9
of itself (float16: 2^-10) where it is small, so that saturated units keep their gradients.  The same call repeats its bits.

The planes of a float32 row hold its elements down to 2^-17 of its largest in 22 bits, smaller ones to 2^-39 of the largest, and no
infinity: where the tensor cores run (above a few rows) a row of x that holds one gives NaN in its row of the result, a row of W
in its column, a row of the gradient in its row of x's gradient.  The 16-bit types keep infinities.

CUDA tensors only; there is no fallback.  The reference's counterpart is ``F.linear`` (src/gru_qat/gru_cell.py:410-435), without
activation and residual.
"""

from __future__ import annotations

import ctypes
from typing import Any, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._scan_common import require_cuda, transformed
from .scan_gated import DTYPES, call_on, rows_contiguous

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "sigmoid": 4, "tanh": 5}


def _check(x, W, bias, residual, activation):
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}; got {activation!r}")
    dtype = x.dtype
    if dtype not in DTYPES:
        raise ValueError(f"x dtype must be float32, bfloat16 or float16; got {dtype}")
    for name, t in (("W", W), ("bias", bias), ("residual", residual)):
        if t is not None and t.dtype != dtype:
            raise ValueError(f"{name} dtype must be x's, {dtype}; got {t.dtype}")
    lead, w = x.shape, W.shape
    if len(w) != 2 or len(lead) < 1 or lead[-1] != w[1]:
        raise ValueError(f"linear_act needs x[..., K] and W[N, K]; got {tuple(lead)} and {tuple(w)}")
    N, K = w
    if N == 0 or K == 0:
        raise ValueError(f"N and K must be > 0; got N={N}, K={K}")
    if x.numel() // K > 2 ** 31 - 512 or N > 2 ** 30 - 16 or K > 2 ** 30 - 16:
        raise ValueError(f"at most 2^31 - 512 rows and 2^30 - 16 columns; got x {tuple(lead)}, W {tuple(w)}")
    if bias is not None and bias.shape != (N,):
        raise ValueError(f"bias shape must be (N,)=({N},); got {tuple(bias.shape)}")
    if residual is not None and residual.shape != (*lead[:-1], N):
        raise ValueError(f"residual shape must be {(*lead[:-1], N)}; got {tuple(residual.shape)}")
    device = x.device
    if not x.is_cuda or any(t is not None and t.device != device for t in (W, bias, residual)):
        given = {k: v for k, v in (("x", x), ("W", W), ("bias", bias), ("residual", residual)) if v is not None}
        require_cuda(**given)
        for name, t in given.items():
            if t.device != device:
                raise ValueError(f"{name} is on {t.device}, x on {device}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as a matrix of rows, in place where its strides allow it."""
    return rows_contiguous(t if t.dim() == 2 else t.reshape(-1, t.shape[-1]))


def _fill(x, W, activation) -> _lib.CLinearArgs:
    a = _lib.CLinearArgs()
    a.M, a.K = x.shape
    a.N = W.shape[0]
    a.dtype, a.activation = DTYPES[x.dtype], ACTIVATIONS[activation]
    a.x, a.ldx, a.W, a.ldw = x.data_ptr(), x.stride(0), W.data_ptr(), W.stride(0)
    return a


_WORKSPACE_TOO_SMALL = 4


def _run(a, backward: bool, x) -> None:
    device = x.device
    lib = _lib.load()
    call = lib.b200gru_linear_act_backward if backward else lib.b200gru_linear_act_forward
    ref = ctypes.byref(a)
    rc = _WORKSPACE_TOO_SMALL if a.dtype == 0 and a.M > 8 else call_on(device, call, ref)
    if rc == _WORKSPACE_TOO_SMALL:                     # 16-bit tensors in the common layout need none, planes of fp32 always
        n = lib.b200gru_linear_act_workspace_bytes(ref, int(backward))
        ws = x.new_empty(n, dtype=torch.uint8)
        a.workspace, a.workspace_bytes = ws.data_ptr(), n
        rc = call_on(device, call, ref)
    if rc:
        _lib._raise(rc, "linear_act backward" if backward else "linear_act")
    _lib._after_call()


def _forward(x, W, bias, residual, activation, want_slope: bool):
    """(y[M, N], slope or None)."""
    lead, N = x.shape[:-1], W.shape[0]
    x, W = _rows(x), rows_contiguous(W)
    M = x.shape[0]
    y = x.new_empty((M, N))
    slope = None
    if want_slope and activation != "none":
        # rows padded to eight elements: 16-byte accesses at any width
        slope = x.new_empty((M, -(-N // 8) * 8), dtype=torch.float32 if x.dtype == torch.float32 else torch.int16)
    if M:
        a = _fill(x, W, activation)
        if bias is not None:
            bias = rows_contiguous(bias)
            a.bias = bias.data_ptr()
        if residual is not None:
            residual = _rows(residual)
            a.residual, a.ldr = residual.data_ptr(), residual.stride(0)
        a.y, a.ldy = y.data_ptr(), N
        if slope is not None:
            a.slope, a.lds = slope.data_ptr(), slope.stride(0)
        _run(a, False, x)
    return (y if len(lead) == 1 else y.reshape(*lead, N)), slope


class LinearActFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x, W, bias, residual, activation):
        y, slope = _forward(x, W, bias, residual, activation, True)
        ctx.save_for_backward(x, W, *([slope] if slope is not None else []))
        ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dy):
        x, W, *slope = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dx = x.new_empty(x.shape) if need_x else None
        M, (N, K) = x.numel() // x.shape[-1], W.shape
        fresh = x.new_empty if M else x.new_zeros
        dW = fresh((N, K)) if need_w else None
        db = fresh((N,)) if need_b else None
        if M and (need_x or need_w or need_b):
            x2, W2, dy2 = _rows(x), rows_contiguous(W), _rows(dy)
            a = _fill(x2, W2, ctx.activation)
            a.dy, a.lddy = dy2.data_ptr(), dy2.stride(0)
            if slope:
                a.slope, a.lds = slope[0].data_ptr(), slope[0].stride(0)
            for name, t in (("dx", dx), ("dW", dW), ("db", db)):
                if t is not None:
                    setattr(a, name, t.data_ptr())
            _run(a, True, x)
        return dx, dW, db, (dy if need_r else None), None


def linear_act(x: torch.Tensor, W: torch.Tensor, bias: Optional[torch.Tensor] = None, *, activation: str = "none",
               residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(x[..., K] @ W[N, K]^T + bias[N]) + residual[..., N]`` in x's type; differentiable in all four tensors.

    ``activation``: none, relu, silu, gelu (the error-function form), sigmoid or tanh.  Rows may have any stride; a
    residual has the result's shape (``expand`` a broadcast one).  Reverse mode only: forward-mode AD and ``torch.func``
    transforms raise an error."""
    _check(x, W, bias, residual, activation)
    if (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, W, bias, residual))) or transformed():
        return LinearActFunction.apply(x, W, bias, residual, activation)
    return _forward(x, W, bias, residual, activation, False)[0]
