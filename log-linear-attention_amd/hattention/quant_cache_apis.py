"""Attention over a cache of keys and values in 8 bits (MI355X): prompts, drafts, decode.

The global attention of a hybrid stack, next to the log-linear scans and ``sliding_apis``: a
cache that keeps every token, in half the memory of 16 bits, which bounds decoding.  The kernels are
libhattn_hip.so's ``hattn_quant_cache_append`` / ``_read`` / ``_attention`` / ``_step``.  No
counterpart in the reference.
"""
import ctypes
import functools
from typing import Optional, Tuple

import torch

from hattention import _lib
from hattention.recurrence_apis import check_lengths

BLOCK = 64
MAX_CAPACITY = 2 ** 30
E4M3 = torch.float8_e4m3fn


_Strides3, _Strides6, _Strides9 = (ctypes.c_longlong * n for n in (3, 6, 9))


def _lead(t):
    """t, or a copy, with contiguous rows that start on 16 bytes, and its batch, token and head
    strides (0 where there is one element: torch leaves such a stride at any value)."""
    n = t.shape
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        row = n[-2] * n[-1]
        return t, (row, 0, n[-1]) if len(n) == 3 else (n[1] * row, row, n[-1])
    s = t.stride()
    if len(n) == 3:  # one token a row
        lead = s[0] if n[0] > 1 else 0, 0, s[1] if n[1] > 1 else 0
    else:
        lead = s[0] if n[0] > 1 else 0, s[1] if n[1] > 1 else 0, s[2] if n[2] > 1 else 0
    if s[-1] == 1 and t.data_ptr() % 16 == 0 and (lead[0] | lead[1] | lead[2]) % 8 == 0:
        return t, lead
    return _lead(t.clone(memory_format=torch.contiguous_format))


@functools.lru_cache(maxsize=256)
def _attention_bytes(*sizes) -> int:
    return _lib.load().hattn_quant_cache_attention_workspace(*sizes)


class QuantCache:
    """The cache of a batch: ``k``, ``v`` [B, G, capacity, D] in e4m3 (``torch.float8_e4m3fn``),
    ``k_scale``, ``v_scale`` [B, G, capacity / 64] fp32 and ``counts`` [B] int32, the tokens that each row
    has had.  Token s of a row is its code times the scale of block s // 64.

    A scale is a power of two, the least for which 448 times it holds every finite value of the
    block (from 2 ** -100 to 2 ** 119, 2 ** 7 for fp16; larger values become 448 times that), so
    that a value has one rounding, of at most 2 ** -4 of itself (2 ** -10 of the scale where that is
    more); infinities and NaN are stored as NaN.  A block whose later tokens are larger gets a larger
    scale, which rounds its older tokens again only where their codes fall below 2 ** -6.

    All five are advanced in place, on the device.  A count may be set back (to drop drafted
    tokens, or to 0 to take a row into use again): the scale of the block that it then ends in stays what
    the dropped tokens made it, and so do the codes of those before them (to go back exactly, keep that
    block's codes and scales).  Tokens past the capacity are counted but not stored, and
    attention gives NaN for such a row."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "counts", "_layout")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor,
                 v_scale: torch.Tensor, counts: torch.Tensor) -> None:
        self.k, self.v, self.k_scale, self.v_scale, self.counts = k, v, k_scale, v_scale, counts
        self._layout = None
        self._check()
        if (k.data_ptr() | v.data_ptr()) % 16:
            raise ValueError("the cache must be aligned to 16 bytes")

    def _check(self) -> None:
        """That the tensors are what the kernels take: in each call, since the attributes can be set.
        A layout that has passed is compared as a whole (0.7 us)."""
        k, v, k_scale, v_scale, counts = self._tensors()
        layout = (k.shape, v.shape, k_scale.shape, v_scale.shape, counts.shape, k.dtype, v.dtype,
                  k_scale.dtype, v_scale.dtype, counts.dtype, k.is_contiguous(), v.is_contiguous(),
                  k_scale.is_contiguous(), v_scale.is_contiguous(), counts.is_contiguous(),
                  k.device, v.device, k_scale.device, v_scale.device, counts.device)
        if layout == self._layout:
            return
        if k.dim() != 4 or k.shape != v.shape or 0 in k.shape or k.shape[2] % BLOCK != 0 or \
                k_scale.shape != (*k.shape[:2], k.shape[2] // BLOCK) or \
                v_scale.shape != k_scale.shape or counts.shape != k.shape[:1]:
            raise ValueError(f"cache of shapes {tuple(k.shape)}, {tuple(v.shape)}, "
                             f"{tuple(k_scale.shape)}, {tuple(v_scale.shape)}, {tuple(counts.shape)}")
        if k.dtype != E4M3 or v.dtype != E4M3 or k_scale.dtype != torch.float32 or \
                v_scale.dtype != torch.float32 or counts.dtype != torch.int32:
            raise ValueError("k and v must be float8_e4m3fn, the scales float32, counts int32")
        if not all(layout[10:15]):
            raise ValueError("the cache must be contiguous: it is advanced in place")
        if k.shape[3] % 16 != 0 or k.shape[3] > 128:
            raise NotImplementedError(f"D={k.shape[3]} is not a multiple of 16 up to 128")
        if k.shape[2] > MAX_CAPACITY:
            raise NotImplementedError(f"capacity={k.shape[2]} above {MAX_CAPACITY}")
        if len(set(layout[15:])) > 1:
            raise RuntimeError("the cache's tensors are on different devices")
        self._layout = layout

    @classmethod
    def empty(cls, B: int, G: int, D: int, capacity: int, device="cuda") -> "QuantCache":
        """A cache without tokens, of at least ``capacity`` (a multiple of 64)."""
        if capacity < 1:
            raise ValueError(f"capacity={capacity}")
        slots = -(-capacity // BLOCK) * BLOCK
        k, v = (torch.zeros(B, G, slots, D, dtype=torch.uint8, device=device).view(E4M3)
                for _ in range(2))
        ks, vs = (torch.ones(B, G, slots // BLOCK, dtype=torch.float32, device=device)
                  for _ in range(2))
        return cls(k, v, ks, vs, torch.zeros(B, dtype=torch.int32, device=device))

    @property
    def capacity(self) -> int:
        return self.k.shape[2]

    def _tensors(self):
        return self.k, self.v, self.k_scale, self.v_scale, self.counts

    def _ptrs(self):
        return (self.k.data_ptr(), self.v.data_ptr(), self.k_scale.data_ptr(),
                self.v_scale.data_ptr(), self.counts.data_ptr())


def _check_half(*tensors) -> None:
    dtype = tensors[0].dtype
    for t in tensors:
        if t.dtype is not dtype:
            raise ValueError("q, k and v must have one dtype")
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise NotImplementedError(f"{dtype}: bf16 or fp16 only")


def _check_new(cache, k, v, lead) -> None:
    B, G, _, D = cache.k.shape
    if k.shape != v.shape or k.shape != (B, *lead, G, D):
        raise ValueError(f"k {tuple(k.shape)}, v {tuple(v.shape)} for a cache {tuple(cache.k.shape)}")


def _check_queries(cache, q, scale) -> float:
    B, G, _, D = cache.k.shape
    H = q.shape[-2]
    if q.shape[0] != B or q.shape[-1] != D:
        raise ValueError(f"q {tuple(q.shape)} for a cache {tuple(cache.k.shape)}")
    if 0 in q.shape:
        raise ValueError("empty tensor")
    if H % G != 0:
        raise ValueError(f"H={H} is not a multiple of G={G}")
    if scale is None:
        scale = D ** -0.5
    elif not 0.0 < scale <= 1e30:
        raise ValueError("scale must be positive and finite")
    return scale


def quant_cache_append(cache: QuantCache, k: torch.Tensor, v: torch.Tensor,
                       lengths: Optional[torch.Tensor] = None) -> QuantCache:
    """Tokens k, v [B, T, G, D] (bf16 or fp16, any strides) enter the cache after each row's last
    one; with ``lengths`` [B] (int32 or int64, on the device) the first lengths[b] of row b.  Keys enter
    with their positions applied.  Returns the cache, advanced in place; a captured call can be
    replayed (the counts are on the device)."""
    cache._check()
    if k.dim() != 4 or 0 in k.shape:
        raise ValueError("k and v must be [B, T, G, D], not empty")
    B, T = k.shape[:2]
    _check_new(cache, k, v, (T,))
    _check_half(k, v)
    if T > cache.capacity:
        raise ValueError(f"T={T} tokens for a capacity of {cache.capacity}")
    dev = _lib.require_device(cache.k, k, v)
    lengths = check_lengths(lengths, B, dev)
    (k, sk), (v, sv) = _lead(k), _lead(v)
    _lib.launch(dev, _lib.load().hattn_quant_cache_append, k.data_ptr(), v.data_ptr(),
                _lib.ptr(lengths), _Strides6(*sk, *sv), *cache._ptrs(), B, T, k.shape[2], k.shape[3],
                cache.capacity, _lib.dtype_code(k))
    _lib.advanced(*cache._tensors())
    return cache


def quant_cache_read(cache: QuantCache, dtype: torch.dtype = torch.bfloat16, start: int = 0,
                     stop: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Tokens start .. stop - 1 (to the capacity without ``stop``) of every row as k, v
    [B, stop - start, G, D] in bf16, fp16 or fp32, as :func:`quant_cache_append` took them; zero where a row
    has none."""
    cache._check()
    B, G, slots, D = cache.k.shape
    stop = slots if stop is None else stop
    if not 0 <= start < stop <= slots:
        raise ValueError(f"tokens {start} to {stop} of {slots}")
    if dtype not in _lib.DTYPE_CODES:
        raise NotImplementedError(f"unsupported dtype {dtype}")
    dev = _lib.require_device(cache.k)
    k, v = (torch.empty(B, stop - start, G, D, dtype=dtype, device=dev) for _ in range(2))
    _lib.launch(dev, _lib.load().hattn_quant_cache_read, *cache._ptrs(), k.data_ptr(), v.data_ptr(),
                B, G, D, slots, start, stop - start, _lib.DTYPE_CODES[dtype])
    return k, v


def quant_cache_attention(cache: QuantCache, q: torch.Tensor, scale: Optional[float] = None,
                          lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of each row's last tokens over the cache, which holds them already
    (:func:`quant_cache_append`): a prompt, a piece of one, or drafted tokens.

    q [B, T, H, D] (bf16 or fp16, any strides), G dividing H (head h reads group h // (H // G)), with
    positions applied.  With ``lengths`` [B] (int32 or int64, on the device) row b has lengths[b] new
    tokens (clamped to [0, T]), else T: query t sees the tokens up to counts[b] - lengths[b] + t.
    ``scale`` defaults to D ** -0.5.  Returns o [B, T, H, D]: zero for t >= lengths[b] and where a
    query sees nothing, NaN where a row has had more tokens than the capacity.

    Scores, softmax and sums are fp32; the probabilities are rounded to q's dtype between the products.
    Sums have a fixed order.  Without gradients.
    """
    cache._check()
    if q.dim() != 4:
        raise ValueError("q must be [B, T, H, D]")
    scale = _check_queries(cache, q, scale)
    _check_half(q)
    dev = _lib.require_device(cache.k, q)
    B, T, H, D = q.shape
    lengths = check_lengths(lengths, B, dev)
    q, sq = _lead(q)
    o = torch.empty(B, T, H, D, dtype=q.dtype, device=dev)
    sizes = B, T, H, cache.k.shape[1], D, cache.capacity
    ws, ws_ptr, ws_bytes = _lib.workspace(_attention_bytes(*sizes), dev)
    _lib.launch(dev, _lib.load().hattn_quant_cache_attention, q.data_ptr(), _lib.ptr(lengths),
                _Strides3(*sq), *cache._ptrs(), o.data_ptr(), *sizes, scale, _lib.dtype_code(q), ws_ptr,
                ws_bytes)
    return o


def quant_cache_step(cache: QuantCache, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                     scale: Optional[float] = None) -> Tuple[torch.Tensor, QuantCache]:
    """One token per row: q [B, H, D], k, v [B, G, D].  The token enters the cache, and q sees it
    and all before it: :func:`quant_cache_append` and :func:`quant_cache_attention` of T = 1 in one
    call, with the same results.  Returns (o [B, H, D], cache), the cache advanced in place; a captured step
    can be replayed."""
    cache._check()
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError("q, k and v must be [B, heads, D]")
    scale = _check_queries(cache, q, scale)
    _check_new(cache, k, v, ())
    _check_half(q, k, v)
    dev = _lib.require_device(cache.k, q, k, v)
    B, H, D = q.shape
    (q, sq), (k, sk), (v, sv) = _lead(q), _lead(k), _lead(v)
    o = torch.empty(B, H, D, dtype=q.dtype, device=dev)
    G, slots = cache.k.shape[1:3]
    ws, ws_ptr, ws_bytes = _lib.workspace(_attention_bytes(B, 1, H, G, D, slots), dev)
    _lib.launch(dev, _lib.load().hattn_quant_cache_step, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                _Strides9(*sq, *sk, *sv), *cache._ptrs(), o.data_ptr(), B, H, G, D, slots, scale,
                _lib.dtype_code(q), ws_ptr, ws_bytes)
    _lib.advanced(*cache._tensors())
    return o, cache
