"""Rotary positions of queries and keys (MI355X): training and decode.

What a hybrid stack's attention layers (``sliding_apis``, ``quant_cache_apis``) apply to q and
k before the scores.  One launch for both tensors, forward and backward (libhattn_hip.so:
``hattn_rotary``).  No counterpart in the reference.
"""
import ctypes
import math
from typing import Optional, Tuple

import torch

from hattention import _lib

MAX_D = 512
LAYOUTS = ("half", "interleaved")


def rotary_frequencies(dim: int, base: float = 10000.0, scaling: Optional[str] = None,
                       factor: float = 1.0, original_length: Optional[int] = None,
                       fast: float = 32.0, slow: float = 1.0,
                       device="cuda") -> Tuple[torch.Tensor, float]:
    """(freqs, scale) for :func:`rotary_embedding`: the dim / 2 frequencies base ** (-2 i / dim) in
    radians a token (fp64, on ``device``), for contexts ``factor`` times as long as trained with
    where ``scaling`` is

    * ``"linear"``: positions divided by ``factor``;
    * ``"ntk"``: a base for which the slowest frequency is divided by ``factor`` and the fastest
      stays, base * factor ** (dim / (dim - 2));
    * ``"yarn"`` (Peng et al. 2023, "YaRN: Efficient Context Window Extension of Large Language
      Models"): with r the turns of a frequency within ``original_length`` tokens, frequencies of
      r >= ``fast`` stay, those of r <= ``slow`` are divided by ``factor``, those between are mixed
      of both, linearly in r; scale = 1 + 0.1 log(factor).  In the others scale = 1.
    """
    if dim < 2 or dim % 2 != 0:
        raise ValueError(f"dim={dim} is not a positive even number")
    if not 1.0 < base < math.inf:
        raise ValueError(f"base={base}")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"scaling={scaling!r}")
    if not 1.0 <= factor < math.inf:
        raise ValueError(f"factor={factor} below 1")
    n, scale = dim // 2, 1.0
    if scaling == "ntk":
        if dim == 2:
            raise ValueError("dim=2 has one frequency, which \"ntk\" keeps")
        base = base * factor ** (dim / (dim - 2))
    freqs = [base ** (-2.0 * i / dim) for i in range(n)]
    if scaling == "linear":
        freqs = [f / factor for f in freqs]
    elif scaling == "yarn":
        if original_length is None or original_length < 1:
            raise ValueError("\"yarn\" needs original_length")
        if not 0.0 < slow < fast:
            raise ValueError(f"fast={fast}, slow={slow}")
        for i, f in enumerate(freqs):
            turns = original_length * f / (2.0 * math.pi)
            stay = min(max((turns - slow) / (fast - slow), 0.0), 1.0)
            freqs[i] = f * stay + f / factor * (1.0 - stay)
        scale = 1.0 + 0.1 * math.log(factor)
    return torch.tensor(freqs, dtype=torch.float64, device=device), scale


_Strides = ctypes.c_longlong * 6


def _lead(t):
    """t with a contiguous last dimension, and its batch, token and head strides (0 where there is
    one element: torch leaves such a stride at any value)."""
    s = t.stride()
    if s[-1] != 1 and t.shape[-1] != 1:
        t = t.contiguous()
        s = t.stride()
    n = t.shape
    if len(n) == 3:  # one token a row
        return t, (s[0] if n[0] > 1 else 0, 0, s[1] if n[1] > 1 else 0)
    return t, (s[0] if n[0] > 1 else 0, s[1] if n[1] > 1 else 0, s[2] if n[2] > 1 else 0)


def _launch(q, k, freqs, positions, interleaved, scale, inverse):
    """(q, k) of [B, T, heads, D], or [B, heads, D], turned."""
    q, strides = _lead(q)
    n = q.shape
    B, H, D = n[0], n[-2], n[-1]
    T = n[1] if len(n) == 4 else 1
    qo, ko, G = torch.empty(n, dtype=q.dtype, device=q.device), None, 0
    if k is not None:
        k, more = _lead(k)
        G = k.shape[-2]
        ko = torch.empty(k.shape, dtype=q.dtype, device=q.device)
        strides += more
    pb = pt = per_row = wide = 0
    if positions is not None:
        per_row = positions.dim() == 1
        wide = positions.dtype == torch.int64
        pb = positions.stride(0) if B > 1 else 0
        pt = positions.stride(1) if not per_row and T > 1 else 0
    _lib.launch(q.device, _lib.load().hattn_rotary, q.data_ptr(), _lib.ptr(k), _Strides(*strides),
                qo.data_ptr(), _lib.ptr(ko), freqs.data_ptr(), freqs.dtype == torch.float64,
                _lib.ptr(positions), wide, pb, pt, per_row, B, T, H, G, D, freqs.shape[0], interleaved,
                scale, inverse, _lib.dtype_code(q))
    return qo, ko


def _turn(q, k, *args):
    """:func:`_launch`, differentiable where that is wanted."""
    return (RotaryFunction.apply if _lib.wants_grad(q, k) else _launch)(q, k, *args)


class RotaryFunction(torch.autograd.Function):
    """(q, k) of :func:`rotary_embedding`; the backward turns the gradients back, and can itself be
    differentiated; tangents are turned as their tensors are."""

    @staticmethod
    def forward(ctx, q, k, freqs, positions, interleaved, scale, inverse):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(freqs, positions)
        ctx.cfg = interleaved, scale, inverse
        if _lib.forward_mode():
            ctx.save_for_forward(freqs, positions)
            ctx.q_shape, ctx.k_shape = q.shape, None if k is None else k.shape
        return _launch(q, k, freqs, positions, interleaved, scale, inverse)

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        # of outputs that are tensors the engine takes zeros, not None
        if tq is None:
            tk, _ = _turn(tk, None, *ctx.saved_tensors, *ctx.cfg)
            return torch.zeros(ctx.q_shape, dtype=tk.dtype, device=tk.device), tk
        tq, tk = _turn(tq, tk, *ctx.saved_tensors, *ctx.cfg)
        if tk is None and ctx.k_shape is not None:
            tk = torch.zeros(ctx.k_shape, dtype=tq.dtype, device=tq.device)
        return tq, tk

    @staticmethod
    def backward(ctx, dq, dk):
        freqs, positions = ctx.saved_tensors
        interleaved, scale, inverse = ctx.cfg
        dq = dq if ctx.needs_input_grad[0] else None
        dk = dk if ctx.needs_input_grad[1] else None
        if dq is not None or dk is not None:
            # grad mode is on where the gradient's own gradient is wanted
            turn = RotaryFunction.apply if torch.is_grad_enabled() or _lib.forward_mode() else _launch
            args = freqs, positions, interleaved, scale, not inverse
            if dq is not None:
                dq, dk = turn(dq, dk, *args)
            else:
                dk, _ = turn(dk, None, *args)
        return dq, dk, None, None, None, None, None


def rotary_embedding(q: torch.Tensor, k: Optional[torch.Tensor], freqs: torch.Tensor,
                     positions: Optional[torch.Tensor] = None, layout: str = "half",
                     scale: float = 1.0) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """q and k turned by their positions: in each head, pair i of the first 2 * len(freqs)
    elements is rotated by position * freqs[i] and multiplied by ``scale``; the others stay.

    q [B, T, H, D] and k [B, T, G, D] (or None), or one token a row, [B, H, D] and [B, G, D], in bf16,
    fp16 or fp32, of any strides; D <= 512.  freqs [n], fp32 or fp64 (:func:`rotary_frequencies`);
    2 n <= D.  ``layout`` "half" pairs elements i and i + n, "interleaved" 2 i and 2 i + 1.
    ``positions`` (int32 or int64, on the device): [B], of each row's first token, or [B, T], of every
    token; None: 0 to T - 1 (one token a row needs [B]).  Returns (q, k), contiguous; gradients
    reach q and k, and so do tangents of forward mode; ``freqs`` that require a gradient are refused.

    Angles are taken and reduced in 64 bits, sines and products in 32, at any position.
    """
    if layout not in LAYOUTS:
        raise ValueError(f"layout={layout!r}: one of {LAYOUTS}")
    one = q.dim() == 3
    if q.dim() not in (3, 4) or (k is not None and k.dim() != q.dim()):
        raise ValueError("q and k must be [B, T, heads, D] or [B, heads, D]")
    if k is not None and (k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1]):
        raise ValueError(f"shapes of q {tuple(q.shape)}, k {tuple(k.shape)}")
    if 0 in q.shape or (k is not None and 0 in k.shape):
        raise ValueError("empty tensor")
    if k is not None and k.dtype != q.dtype:
        raise ValueError("q and k must have one dtype")
    _lib.dtype_code(q)
    D = q.shape[-1]
    if freqs.dim() != 1 or not 1 <= freqs.shape[0] <= D // 2:
        raise ValueError(f"freqs {tuple(freqs.shape)} for heads of {D}")
    if freqs.dtype not in (torch.float32, torch.float64):
        raise NotImplementedError(f"freqs in {freqs.dtype}")
    if _lib.wants_grad(freqs):
        raise NotImplementedError("freqs have no gradient: pass them detached")
    if D > MAX_D:
        raise NotImplementedError(f"D={D} above {MAX_D}")
    if not math.isfinite(scale) or abs(scale) > 1e30:
        raise ValueError(f"scale={scale}")
    if positions is not None:
        if positions.shape != q.shape[:1] and (one or positions.shape != q.shape[:2]):
            raise ValueError(f"positions {tuple(positions.shape)} for q {tuple(q.shape)}")
        if positions.dtype not in (torch.int32, torch.int64):
            raise NotImplementedError(f"positions in {positions.dtype}")
    elif one:
        raise ValueError("one token a row needs positions [B]")
    _lib.require_device(q, k, freqs, positions)
    if not freqs.is_contiguous():
        freqs = freqs.contiguous()
    return _turn(q, k, freqs, positions, layout == "interleaved", float(scale), False)
