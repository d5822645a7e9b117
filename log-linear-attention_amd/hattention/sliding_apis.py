"""Sliding-window attention with sinks (MI355X): training, prefill and decode.

The local attention of a hybrid stack, next to the log-linear scans (whose entry points
``hattention_kernel`` / ``hattention_prefill`` / ``hattention_step`` it follows): query t
sees the ``window`` keys that end with its own, and the first ``sinks`` tokens.  The
kernels are libhattn_hip.so's ``hattn_sliding_fwd`` / ``_bwd`` / ``_cache_fill`` /
``_step``.  No counterpart in the reference.
"""
import ctypes
import functools
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from hattention import _lib
from hattention.recurrence_apis import check_lengths

MAX_SINKS = 64


@functools.lru_cache(maxsize=256)
def _step_bytes(*sizes) -> int:
    return _lib.load().hattn_sliding_step_workspace(*sizes)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t where its rows start on 16 bytes and are contiguous, else a copy that does."""
    if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and \
            all(s % 8 == 0 for n, s in zip(t.shape[:-1], t.stride()) if n > 1) and \
            t.stride(1) < 2 ** 24:
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _strides(*tensors):
    """Batch, token and head strides of each tensor, for the C-ABI (0 where the size is 1:
    torch leaves such a stride at any value)."""
    s = [x if n > 1 else 0 for t in tensors for n, x in zip(t.shape[:3], t.stride())]
    return (ctypes.c_longlong * len(s))(*s)


def _check_shapes(q, k, v, window, sinks, scale):
    """The scale; q [.., H, D], k, v [.., G, D]."""
    if k.shape != v.shape or q.shape[:-2] != k.shape[:-2] or q.shape[-1] != k.shape[-1]:
        raise ValueError(f"shapes of q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if 0 in q.shape or 0 in k.shape:
        raise ValueError("empty tensor")
    H, D = q.shape[-2:]
    G = k.shape[-2]
    if H % G != 0:
        raise ValueError(f"H={H} is not a multiple of G={G}")
    if window < 1 or sinks < 0:
        raise ValueError(f"window={window}, sinks={sinks}")
    if scale is None:
        scale = D ** -0.5
    elif not 0.0 < scale <= 1e30:
        raise ValueError("scale must be positive and finite")
    if q.dtype != k.dtype or q.dtype != v.dtype:
        raise ValueError("q, k and v must have one dtype")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise NotImplementedError(f"{q.dtype}: bf16 or fp16 only")
    if sinks > MAX_SINKS:
        raise NotImplementedError(f"sinks={sinks} above {MAX_SINKS}")
    if D % 8 != 0 or D > 128:
        raise NotImplementedError(f"D={D} is not a multiple of 8 up to 128")
    return scale


def _forward(q, k, v, lengths, window, sinks, scale, keep):
    """(o, lse or None)."""
    B, T, H, D = q.shape
    dev = q.device
    o = torch.empty(B, T, H, D, dtype=q.dtype, device=dev)
    lse = torch.empty(B, H, T, dtype=torch.float32, device=dev) if keep else None
    _lib.launch(dev, _lib.load().hattn_sliding_fwd, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                _lib.ptr(lengths), _strides(q, k, v), o.data_ptr(), _lib.ptr(lse), B, T, H,
                k.shape[2], D, window, sinks, scale, _lib.dtype_code(q))
    return o, lse


class SlidingWindowFunction(torch.autograd.Function):
    """o of :func:`sliding_window_attention`; the backward makes the scores again."""

    @staticmethod
    def forward(ctx, q, k, v, lengths, window, sinks, scale):
        o, lse = _forward(q, k, v, lengths, window, sinks, scale, True)
        ctx.save_for_backward(q, k, v, lengths, o, lse)
        ctx.cfg = window, sinks, scale
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, lengths, o, lse = ctx.saved_tensors
        window, sinks, scale = ctx.cfg
        B, T, H, D = q.shape
        G = k.shape[2]
        dev = q.device
        do = do.contiguous()
        do = do if do.data_ptr() % 16 == 0 else do.clone()
        dq = torch.empty(B, T, H, D, dtype=q.dtype, device=dev)
        dk, dv = (torch.empty(B, T, G, D, dtype=q.dtype, device=dev) for _ in range(2))
        lib = _lib.load()
        ws, ws_ptr, ws_bytes = _lib.workspace(
            lib.hattn_sliding_bwd_workspace(B, T, H, G, D, window, sinks), dev)
        _lib.launch(dev, lib.hattn_sliding_bwd, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                    _lib.ptr(lengths), _strides(q, k, v), o.data_ptr(), lse.data_ptr(),
                    do.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), B, T, H, G, D,
                    window, sinks, scale, _lib.dtype_code(q), ws_ptr, ws_bytes)
        need = ctx.needs_input_grad
        return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None,
                None, None, None, None)


def sliding_window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int,
                             sinks: int = 0, scale: Optional[float] = None,
                             lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention over a window and the first tokens.

    q [B, T, H, D], k, v [B, T, G, D] in bf16 or fp16, G dividing H (head h reads group
    h // (H // G)), D a multiple of 8 up to 128; any strides (views whose rows start on 16
    bytes are read in place).  Query t sees key s where s <= t and (t - s < window or
    s < sinks); sinks <= 64.  ``scale`` defaults to D ** -0.5.  ``lengths`` [B] (int32 or
    int64, on the device) are the tokens of each row of a padded batch: outputs and
    gradients past them are zero, inputs past them are not used.  Returns o [B, T, H, D].

    Scores, softmax and sums are fp32; the probabilities and the gradients of the scores are
    rounded to the inputs' dtype between the products.  Gradients are summed in a fixed order.
    """
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q, k and v must be [B, T, heads, D]")
    scale = _check_shapes(q, k, v, window, sinks, scale)
    dev = _lib.require_device(q, k, v)
    lengths = check_lengths(lengths, q.shape[0], dev)
    q, k, v = _rows(q), _rows(k), _rows(v)
    window = min(window, q.shape[1])  # a window of T keys holds every earlier one
    if _lib.wants_grad(q, k, v):
        return SlidingWindowFunction.apply(q, k, v, lengths, window, sinks, scale)
    return _forward(q, k, v, lengths, window, sinks, scale, False)[0]


class SlidingState:
    """The cache of a decoding batch: ``k``, ``v`` [B, G, sinks + window, D] and ``counts``
    [B] int32, the tokens that each row has seen.  Slot s < sinks holds token s, slot
    sinks + i the last token p >= sinks with p - sinks = i modulo window.  The step advances
    all three in place, on the device."""

    __slots__ = ("k", "v", "counts", "window", "sinks", "_layout")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, counts: torch.Tensor, window: int,
                 sinks: int) -> None:
        self.k, self.v, self.counts, self.window, self.sinks = k, v, counts, window, sinks
        self._layout = None
        self._check()
        if (k.data_ptr() | v.data_ptr()) % 16:
            raise ValueError("the cache must be aligned to 16 bytes")

    def _check(self) -> None:
        """That the tensors are what the kernel takes: in each step, since the attributes can be set.
        A layout that has passed is compared as a whole."""
        k, v, counts, window, sinks = self.k, self.v, self.counts, self.window, self.sinks
        layout = (k.shape, v.shape, counts.shape, k.dtype, v.dtype, counts.dtype, k.is_contiguous(),
                  v.is_contiguous(), counts.is_contiguous(), window, sinks)
        if layout == self._layout:
            return
        if k.dim() != 4 or k.shape != v.shape or k.shape[2] != sinks + window or \
                counts.shape != (k.shape[0],):
            raise ValueError(f"cache of shapes {tuple(k.shape)}, {tuple(v.shape)}, "
                             f"{tuple(counts.shape)} for window={window}, sinks={sinks}")
        if k.dtype != v.dtype or counts.dtype != torch.int32:
            raise ValueError("k and v must have one dtype and counts be int32")
        if not (k.is_contiguous() and v.is_contiguous() and counts.is_contiguous()):
            raise ValueError("the cache must be contiguous: it is advanced in place")
        self._layout = layout

    @classmethod
    def empty(cls, B: int, G: int, D: int, window: int, sinks: int = 0,
              dtype: torch.dtype = torch.bfloat16, device="cuda") -> "SlidingState":
        """A cache that has seen no token."""
        k, v = (torch.zeros(B, G, sinks + window, D, dtype=dtype, device=device)
                for _ in range(2))
        return cls(k, v, torch.zeros(B, dtype=torch.int32, device=device), window, sinks)


@torch.no_grad()
def sliding_window_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int,
                           sinks: int = 0, scale: Optional[float] = None,
                           lengths: Optional[torch.Tensor] = None
                           ) -> Tuple[torch.Tensor, SlidingState]:
    """:func:`sliding_window_attention` of a batch of prompts, without gradients, and the
    cache that decoding goes on from.  Returns (o, state)."""
    o = sliding_window_attention(q, k, v, window, sinks, scale, lengths)
    B, T, G, D = k.shape
    dev = k.device
    k, v = _rows(k), _rows(v)
    lengths = check_lengths(lengths, B, dev)
    kc, vc = (torch.empty(B, G, sinks + window, D, dtype=k.dtype, device=dev) for _ in range(2))
    counts = torch.empty(B, dtype=torch.int32, device=dev)
    _lib.launch(dev, _lib.load().hattn_sliding_cache_fill, k.data_ptr(), v.data_ptr(),
                _lib.ptr(lengths), _strides(k, v), kc.data_ptr(), vc.data_ptr(),
                counts.data_ptr(), B, T, G, D, window, sinks, _lib.dtype_code(k))
    return o, SlidingState(kc, vc, counts, window, sinks)


@torch.no_grad()
def sliding_window_step(state: SlidingState, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                        scale: Optional[float] = None) -> Tuple[torch.Tensor, SlidingState]:
    """One token per row: q [B, H, D], k, v [B, G, D].  The token enters the cache, and q
    sees it, the window before it and the sinks.  Returns (o [B, H, D], state), the state
    advanced in place; a captured step can be replayed (the counts are on the device)."""
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("q, k and v must be [B, heads, D]")
    state._check()
    window, sinks, kc = state.window, state.sinks, state.k
    scale = _check_shapes(q, k, v, window, sinks, scale)
    B, H, D = q.shape
    G = k.shape[1]
    if kc.shape != (B, G, sinks + window, D) or kc.dtype != q.dtype:
        raise ValueError(f"cache {tuple(kc.shape)} in {kc.dtype} for k {tuple(k.shape)} in {k.dtype}")
    dev = _lib.require_device(q, k, v, kc, state.v, state.counts)
    q, k, v = (t if t.is_contiguous() and t.data_ptr() % 16 == 0
               else t.clone(memory_format=torch.contiguous_format) for t in (q, k, v))
    o = torch.empty_like(q)
    ws, ws_ptr, ws_bytes = _lib.workspace(_step_bytes(B, H, G, D, window, sinks), dev)
    _lib.launch(dev, _lib.load().hattn_sliding_step, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                kc.data_ptr(), state.v.data_ptr(), state.counts.data_ptr(), o.data_ptr(), B, H, G,
                D, window, sinks, scale, _lib.dtype_code(q), ws_ptr, ws_bytes)
    _lib.advanced(kc, state.v, state.counts)
    return o, state
