"""Gated linear recurrence: the GRU update with gates from the input alone.

    z = sigmoid(x)    n = tanh(c) (or c)    h_t = z * h_{t-1} + (1 - z) * n        gi[t, b] = (x[H], c[H])

Without hidden weights a step is an affine map of the state, so the scan is not a chain of T dependent
steps: time is cut into tiles whose maps are joined in a fixed order.  ``gated_scan`` runs whole
sequences and has gradients; ``gated_step`` advances a served batch by one token.

Sequences of a batch may have lengths of their own.  Behind the last step of a row nothing is read into
its results (whatever the padding holds), ``out`` and the gradient of ``gi`` are zero, and ``h_T`` is
the state after its last step.  Lengths outside [0, T] count as the nearer end.

Element types float32, bfloat16 and float16; states (``h0``, ``h_T``) are float32 in all of them, and so
is everything inside: a state is exact to float32 rounding for the gates that came in, a gate to a few units of itself whether it is
open or closed.  (Gates of 16 bits carry their own rounding into it.)  The same call repeats its bits.  CUDA tensors only; there is no fallback.  No
counterpart in the reference, whose recurrences all have hidden weights (scan_diagonal.py:79-124).
"""

from __future__ import annotations

import ctypes
from typing import Any, Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._scan_common import require_cuda, transformed

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_CANDIDATES = {"identity": 0, "tanh": 1}


def call_on(device: torch.device, fn, *args) -> int:
    """``fn(*args, stream)`` on the device's current stream, with that device current.  (The raw handles: a token's call
    takes longer on the host than on the GPU, and the stream object alone was a sixth of it.)"""
    index = device.index
    if torch._C._cuda_getDevice() == index:
        return fn(*args, torch._C._cuda_getCurrentRawStream(index))
    with torch.cuda.device(device):
        return fn(*args, torch._C._cuda_getCurrentRawStream(index))


def rows_contiguous(t: torch.Tensor) -> torch.Tensor:
    """``t`` itself where its last axis is contiguous (any other strides), else a copy."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _check_common(gi, candidate, dims, layout) -> Tuple[int, ...]:
    if not isinstance(gi, torch.Tensor):
        raise ValueError("gi must be a tensor")
    if candidate not in _CANDIDATES:
        raise ValueError(f"candidate must be 'tanh' or 'identity'; got {candidate!r}")
    if gi.dtype not in DTYPES:
        raise ValueError(f"gi dtype must be float32, bfloat16 or float16; got {gi.dtype}")
    shape = gi.shape
    if len(shape) != dims or shape[-1] % 2 != 0:
        raise ValueError(f"gi must be {layout}; got {tuple(shape)}")
    return shape


def _check_state(name, h, B, H):
    if h.dtype != torch.float32:
        raise ValueError(f"{name} dtype must be float32; got {h.dtype}")
    if h.shape != (B, H):
        raise ValueError(f"{name} shape must be (B, H)=({B}, {H}); got {tuple(h.shape)}")


def _check_size(T, B, H):
    if T > 2 ** 30 or H > 2 ** 30 - 64 or B * H > 2 ** 31 - 1:
        raise ValueError(f"at most 2^30 steps, 2^30 - 64 units and 2^31 - 1 states; got T={T}, B={B}, H={H}")


def _check_devices(gi, names, others):
    if not gi.is_cuda or any(t is not None and t.device != gi.device for t in others):
        given = {n: t for n, t in zip(names, others) if t is not None}
        require_cuda(gi=gi, **given)
        for name, t in given.items():
            if t.device != gi.device:
                raise ValueError(f"{name} is on {t.device}, gi on {gi.device}")


def _check_scan(gi, h0, lengths, candidate) -> None:
    T, B, two_h = _check_common(gi, candidate, 3, "[T, B, 2H]")
    H = two_h // 2
    if T == 0 or B == 0 or H == 0:
        raise ValueError(f"T, B and H must be > 0; got T={T}, B={B}, H={H}")
    _check_size(T, B, H)
    if h0 is not None:
        _check_state("h0", h0, B, H)
    if lengths is not None:
        if lengths.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"lengths dtype must be int32 or int64; got {lengths.dtype}")
        if lengths.shape != (B,):
            raise ValueError(f"lengths shape must be (B,)=({B},); got {tuple(lengths.shape)}")
    _check_devices(gi, ("h0", "lengths"), (h0, lengths))


def _empty_like_rows(gi: torch.Tensor, cols: int) -> torch.Tensor:
    """``[T, B, cols]`` in gi's order of axes (a batch-first view stays one)."""
    T, B, _ = gi.shape
    if gi.stride(0) < gi.stride(1):
        return gi.new_empty((B, T, cols)).transpose(0, 1)
    return gi.new_empty((T, B, cols))


def _fill(gi, h0, lengths, candidate) -> _lib.CGatedArgs:
    a = _lib.CGatedArgs()
    a.T, a.B, two_h = gi.shape
    a.H = two_h // 2
    a.dtype, a.candidate_tanh = DTYPES[gi.dtype], _CANDIDATES[candidate]
    a.gi = gi.data_ptr()
    a.gi_t, a.gi_b, _ = gi.stride()
    if h0 is not None:
        a.h0, a.h0_b = h0.data_ptr(), h0.stride(0)
    if lengths is not None:
        a.lengths, a.length_bytes = lengths.data_ptr(), lengths.element_size()
    return a


def _forward(gi, h0, lengths, candidate, want_states: bool):
    lib = _lib.load()
    gi = rows_contiguous(gi)
    h0 = None if h0 is None else rows_contiguous(h0)
    lengths = None if lengths is None else lengths.contiguous()
    T, B, H = gi.shape[0], gi.shape[1], gi.shape[2] // 2
    out = _empty_like_rows(gi, H)
    h_T = gi.new_empty((B, H), dtype=torch.float32)
    states = None
    if want_states:
        states = gi.new_empty(lib.b200gru_gated_states_bytes(T, B, H) // 4, dtype=torch.float32)
    a = _fill(gi, h0, lengths, candidate)
    a.out, a.h_T = out.data_ptr(), h_T.data_ptr()
    a.out_t, a.out_b, _ = out.stride()
    if states is not None:
        a.states = states.data_ptr()
    rc = call_on(gi.device, lib.b200gru_gated_scan_forward, ctypes.byref(a))
    if rc:
        _lib._raise(rc, "gated scan forward")
    _lib._after_call()
    return out, h_T, states


def _backward(gi, h0, lengths, candidate, states, dout, dh_T, want_h0: bool):
    lib = _lib.load()
    gi = rows_contiguous(gi)
    lengths = None if lengths is None else lengths.contiguous()
    dgi = _empty_like_rows(gi, gi.shape[2])
    dh0 = gi.new_empty((gi.shape[1], gi.shape[2] // 2), dtype=torch.float32) if want_h0 else None
    a = _fill(gi, None, lengths, candidate)
    a.states = states.data_ptr()
    if dout is not None:
        dout = rows_contiguous(dout)
        a.dout = dout.data_ptr()
        a.dout_t, a.dout_b, _ = dout.stride()
    if dh_T is not None:
        dh_T = rows_contiguous(dh_T)
        a.dh_T, a.dh_b = dh_T.data_ptr(), dh_T.stride(0)
    a.dgi = dgi.data_ptr()
    a.dgi_t, a.dgi_b, _ = dgi.stride()
    if dh0 is not None:
        a.dh0 = dh0.data_ptr()
    rc = call_on(gi.device, lib.b200gru_gated_scan_backward, ctypes.byref(a))
    if rc:
        _lib._raise(rc, "gated scan backward")
    _lib._after_call()
    return dgi, dh0


class GatedScanFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, gi, h0, lengths, candidate):
        out, h_T, states = _forward(gi, h0, lengths, candidate, True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(gi, states, *([lengths] if lengths is not None else []))
        ctx.has_lengths, ctx.candidate = lengths is not None, candidate
        return out, h_T

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dout, dh_T):
        if dout is None and dh_T is None:
            return None, None, None, None
        gi, states = ctx.saved_tensors[:2]
        lengths = ctx.saved_tensors[2] if ctx.has_lengths else None
        dgi, dh0 = _backward(gi, None, lengths, ctx.candidate, states, dout, dh_T, ctx.needs_input_grad[1])
        return (dgi if ctx.needs_input_grad[0] else None), dh0, None, None


def gated_scan(gi: torch.Tensor, h0: Optional[torch.Tensor] = None, *, lengths: Optional[torch.Tensor] = None,
               candidate: str = "tanh") -> Tuple[torch.Tensor, torch.Tensor]:
    """``(out[T, B, H], h_T[B, H])`` of ``gi[T, B, 2H]`` from ``h0`` (zeros where None); differentiable in ``gi`` and ``h0``.

    ``gi`` may have any strides over time and batch (a transposed batch-first tensor is read where it lies, and ``out``
    comes in the same order of axes).  ``lengths``: int32 or int64 ``[B]`` on the same device, read there.  Reverse mode only:
    forward-mode AD and ``torch.func`` transforms raise an error."""
    _check_scan(gi, h0, lengths, candidate)
    if (torch.is_grad_enabled() and (gi.requires_grad or (h0 is not None and h0.requires_grad))) or transformed():
        return GatedScanFunction.apply(gi, h0, lengths, candidate)
    return _forward(gi, h0, lengths, candidate, False)[:2]


def gated_step(gi: torch.Tensor, h: torch.Tensor, *, candidate: str = "tanh",
               out_state: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """One token of every sequence: ``(out[B, H], new state[B, H])`` of ``gi[B, 2H]`` and the state ``h``.

    The new state goes into ``out_state`` where given, which may be ``h`` itself (update in place).  Serving only: it has
    no gradients; ``gated_scan`` of one step has."""
    B, two_h = _check_common(gi, candidate, 2, "[B, 2H]")
    H = two_h // 2
    if B == 0 or H == 0:
        raise ValueError(f"B and H must be > 0; got B={B}, H={H}")
    _check_size(1, B, H)
    _check_state("h", h, B, H)
    if out_state is not None:
        _check_state("out_state", out_state, B, H)
    _check_devices(gi, ("h", "out_state"), (h, out_state))
    if transformed():
        raise ValueError("gated_step is one opaque call: not for function transforms, forward-mode AD or tracing")
    if torch.is_grad_enabled() and (gi.requires_grad or h.requires_grad or (out_state is not None and out_state.requires_grad)):
        raise ValueError("gated_step has no gradients: call it under torch.no_grad(), or gated_scan on gi[None]")
    gi, device = rows_contiguous(gi), gi.device
    if out_state is None:
        h = rows_contiguous(h)
        new = gi.new_empty((B, H), dtype=torch.float32)
    else:
        new = out_state
        if (new.stride(1) != 1 and H > 1) or (B > 1 and new.stride(0) < H):
            raise ValueError(f"out_state must have contiguous rows that do not overlap; got strides {new.stride()}")
        same = new.data_ptr() == h.data_ptr() and new.stride() == h.stride()
        if not same and _overlap(new, h):
            raise ValueError("out_state must be h itself or not overlap it")
        if _overlap(new, gi):
            raise ValueError("out_state must not overlap gi")
        h = h if same else rows_contiguous(h)
    out = gi.new_empty((B, H))
    rc = call_on(device, _lib.load().b200gru_gated_step, DTYPES[gi.dtype], _CANDIDATES[candidate], B, H, gi.data_ptr(),
                 gi.stride(0), h.data_ptr(), h.stride(0), out.data_ptr(), new.data_ptr(), max(new.stride(0), H))
    if rc:
        _lib._raise(rc, "gated step")
    if out_state is not None:
        torch.autograd.graph.increment_version(new)      # autograd refuses what it saved of the old state, as after any in-place write
    return out, new


def _span(t: torch.Tensor) -> Tuple[int, int]:
    first = t.data_ptr()
    return first, first + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the address ranges of two tensors meet, rows interleaved in one another counted as meeting."""
    (a0, a1), (b0, b1) = _span(a), _span(b)
    return a0 < b1 and b0 < a1
