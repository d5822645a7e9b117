"""Gated linear recurrence per channel, ``h_t = exp(g_t) h_{t-1} + x_t`` (MI355X).

The plain recurrent mixer of a hybrid stack, next to the log-linear scans: no keys and
queries, one fp32 state per channel.  Forward and backward each read their inputs once
(libhattn_hip.so: ``hattn_gated_recurrence_fwd`` / ``_bwd`` / ``_step``).  No counterpart
in the reference.
"""
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from hattention import _lib


def check_lengths(lengths, B: int, dev) -> Optional[torch.Tensor]:
    """lengths as a contiguous int32 tensor [B] on ``dev`` (values are clamped on the device)."""
    if lengths is None:
        return None
    if not isinstance(lengths, torch.Tensor) or lengths.shape != (B,):
        raise ValueError(f"lengths must be a tensor of {B} values")
    if lengths.dtype not in (torch.int32, torch.int64):
        raise NotImplementedError(f"lengths in {lengths.dtype}")
    if lengths.device != dev:
        raise RuntimeError("tensors on different devices")
    if lengths.dtype == torch.int64:
        lengths = lengths.clamp(0, 2 ** 31 - 1).to(torch.int32)
    return lengths.contiguous()


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t contiguous and starting on 8 bytes: the kernels read two channels at a time."""
    t = t.contiguous()
    return t if t.data_ptr() % 8 == 0 else t.clone()


def _forward(x, g, h0, lengths, final, keep):
    """(o, ht or None, carry or None)."""
    B, T, D = x.shape
    dev = x.device
    lib = _lib.load()
    code = _lib.dtype_code(x)
    o = torch.empty(B, T, D, dtype=x.dtype, device=dev)
    ht = torch.empty(B, D, dtype=torch.float32, device=dev) if final else None
    carry = torch.empty(B, lib.hattn_gated_recurrence_segments(T, D, code), D, dtype=torch.float32,
                        device=dev) if keep else None
    ws, ws_ptr, ws_bytes = _lib.workspace(lib.hattn_gated_recurrence_workspace(B, T, D, code), dev)
    _lib.launch(dev, lib.hattn_gated_recurrence_fwd, x.data_ptr(), g.data_ptr(), _lib.ptr(h0),
                _lib.ptr(lengths), o.data_ptr(), _lib.ptr(ht), _lib.ptr(carry), B, T, D,
                code, _lib.dtype_code(g), ws_ptr, ws_bytes)
    return o, ht, carry


class GatedRecurrenceFunction(torch.autograd.Function):
    """(o, ht) of :func:`gated_linear_recurrence`.  The states that enter each segment are
    kept for the backward (4 bytes for 128 or 256 tokens of a channel)."""

    @staticmethod
    def forward(ctx, x, g, h0, lengths, final):
        ctx.set_materialize_grads(False)
        o, ht, carry = _forward(x, g, h0, lengths, final, True)
        ctx.save_for_backward(x, g, carry, lengths)
        return o, ht

    @staticmethod
    @once_differentiable
    def backward(ctx, do, dht):
        x, g, carry, lengths = ctx.saved_tensors
        B, T, D = x.shape
        dev = x.device
        if do is None:
            if dht is None:
                return None, None, None, None, None
            do = torch.zeros_like(x)
        do = _aligned(do)
        dht = dht.contiguous() if dht is not None else None
        dx, dg = torch.empty_like(x), torch.empty_like(g)
        dh0 = torch.empty(B, D, dtype=torch.float32, device=dev) \
            if ctx.needs_input_grad[2] else None
        lib = _lib.load()
        code = _lib.dtype_code(x)
        ws, ws_ptr, ws_bytes = _lib.workspace(
            lib.hattn_gated_recurrence_workspace(B, T, D, code), dev)
        _lib.launch(dev, lib.hattn_gated_recurrence_bwd, x.data_ptr(), g.data_ptr(),
                    carry.data_ptr(), _lib.ptr(lengths), do.data_ptr(), _lib.ptr(dht),
                    dx.data_ptr(), dg.data_ptr(), _lib.ptr(dh0), B, T, D, code,
                    _lib.dtype_code(g), ws_ptr, ws_bytes)
        need = ctx.needs_input_grad
        return dx if need[0] else None, dg if need[1] else None, dh0, None, None


def _check_gates(x, g):
    if g.shape != x.shape:
        raise ValueError("x and g must have the same shape")
    _lib.dtype_code(x)
    if g.dtype not in (x.dtype, torch.float32):
        raise NotImplementedError(f"g in {g.dtype} with x in {x.dtype}")


def gated_linear_recurrence(x: torch.Tensor, g: torch.Tensor,
                            initial_state: Optional[torch.Tensor] = None,
                            output_final_state: bool = False,
                            lengths: Optional[torch.Tensor] = None):
    """``o_t = h_t = exp(g_t) h_{t-1} + x_t`` for each channel.

    x [B, T, D] (bf16, fp16 or fp32), g [B, T, D] log-decays in x's dtype or fp32 (-inf
    resets a channel whose state is finite; the product of exp(g) over 256 tokens has to
    stay in fp32's range, as that of decays does), initial_state [B, D] (zero where None), lengths [B] (int32 or
    int64, on the device) the tokens of each row of a padded batch: outputs and gradients
    past them are zero, inputs past them are not used.  Returns o in x's dtype, or with
    ``output_final_state`` ``(o, ht)``, ht [B, D] fp32 the state after each row's last
    token.  States and sums are fp32.
    """
    if x.dim() != 3:
        raise ValueError("x must be [B, T, D]")
    if 0 in x.shape:
        raise ValueError(f"empty x {tuple(x.shape)}")
    _check_gates(x, g)
    B, T, D = x.shape
    if initial_state is not None and initial_state.shape != (B, D):
        raise ValueError(f"initial_state must be [{B}, {D}]")
    dev = _lib.require_device(x, g, initial_state)
    lengths = check_lengths(lengths, B, dev)
    x, g = _aligned(x), _aligned(g)
    h0 = initial_state.float().contiguous() if initial_state is not None else None
    if torch.is_grad_enabled() and (x.requires_grad or g.requires_grad
                                    or (h0 is not None and h0.requires_grad)):
        o, ht = GatedRecurrenceFunction.apply(x, g, h0, lengths, output_final_state)
    else:
        o, ht, _ = _forward(x, g, h0, lengths, output_final_state, False)
    return (o, ht) if output_final_state else o


@torch.no_grad()
def gated_linear_recurrence_step(state: torch.Tensor, x: torch.Tensor, g: torch.Tensor
                                 ) -> Tuple[torch.Tensor, torch.Tensor]:
    """One token: state [B, D] (fp32, contiguous) becomes ``exp(g) state + x`` in place.
    x, g [B, D].  Returns (o [B, D] in x's dtype, state)."""
    if x.dim() != 2:
        raise ValueError("x must be [B, D]")
    _check_gates(x, g)
    if state.shape != x.shape:
        raise ValueError("state must have x's shape")
    if state.dtype != torch.float32:
        raise NotImplementedError(f"state in {state.dtype}: states are fp32")
    if not state.is_contiguous():
        raise ValueError("state must be contiguous: it is advanced in place")
    dev = _lib.require_device(state, x, g)
    x, g = x.contiguous(), g.contiguous()
    o = torch.empty_like(x)
    B, D = x.shape
    _lib.launch(dev, _lib.load().hattn_gated_recurrence_step, state.data_ptr(), x.data_ptr(),
                g.data_ptr(), o.data_ptr(), B, D, _lib.dtype_code(x), _lib.dtype_code(g))
    return o, state
