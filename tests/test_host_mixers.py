"""Refusals of the hybrid stack's mixers and norm: the package's exceptions and the C-ABI's
status codes, on the host, before any launch."""
import ctypes

import pytest
import torch

from hattention import _lib
from hattention.norm_apis import layer_norm
from hattention.recurrence_apis import (check_lengths, gated_linear_recurrence,
                                        gated_linear_recurrence_step)
from hattention.sliding_apis import (SlidingState, sliding_window_attention,
                                     sliding_window_prefill, sliding_window_step)

BF, FS = torch.bfloat16, torch.float32
e = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype)


def raises(kind, fn, *args, **kw):
    with pytest.raises(kind):
        fn(*args, **kw)


def test_layer_norm():
    x = e(3, 16)
    raises(ValueError, layer_norm, torch.zeros((), dtype=BF))
    raises(ValueError, layer_norm, x, e(15))
    raises(ValueError, layer_norm, x, e(16), e(16, 1))
    raises(ValueError, layer_norm, x, e(16), e(16, dtype=FS))
    raises(ValueError, layer_norm, x, residual=e(16))
    raises(ValueError, layer_norm, x, residual=e(3, 1))
    raises(NotImplementedError, layer_norm, x, residual=e(3, 16, dtype=torch.float16))
    raises(NotImplementedError, layer_norm, x.double())
    raises(NotImplementedError, layer_norm, e(1, 16385))
    raises(NotImplementedError, layer_norm, x, e(16, dtype=torch.float64))
    raises(RuntimeError, layer_norm, x)  # not on a HIP device


def test_recurrence():
    x, g = e(2, 3, 4), e(2, 3, 4)
    f = gated_linear_recurrence
    raises(ValueError, f, x[0], g[0])
    raises(ValueError, f, x, g[:, :2])
    raises(ValueError, f, e(2, 0, 4), e(2, 0, 4))
    raises(ValueError, f, x, g, e(2, 3, dtype=FS))
    raises(NotImplementedError, f, x, g.half())
    raises(NotImplementedError, f, x.double(), g.double())
    raises(RuntimeError, f, x, g)
    cpu = torch.device("cpu")
    raises(ValueError, check_lengths, torch.ones(3, dtype=torch.int32), 2, cpu)
    raises(ValueError, check_lengths, [1, 2], 2, cpu)
    raises(NotImplementedError, check_lengths, torch.ones(2), 2, cpu)
    raises(RuntimeError, check_lengths, torch.ones(2, dtype=torch.int32), 2, torch.device("cuda:0"))
    big = check_lengths(torch.tensor([2 ** 40, -3]), 2, cpu)
    assert big.dtype == torch.int32 and big.tolist() == [2 ** 31 - 1, 0]


def test_recurrence_step():
    x, g, h = e(2, 4), e(2, 4), e(2, 4, dtype=FS)
    f = gated_linear_recurrence_step
    raises(ValueError, f, h, x[0], g[0])
    raises(ValueError, f, h, x, g[:1])
    raises(ValueError, f, h[:1], x, g)
    raises(NotImplementedError, f, h.to(BF), x, g)
    raises(ValueError, f, e(4, 2, dtype=FS).t(), x, g)
    raises(RuntimeError, f, h, x, g)


def test_sliding():
    q, k, v = e(2, 5, 4, 64), e(2, 5, 2, 64), e(2, 5, 2, 64)
    for f in (sliding_window_attention, sliding_window_prefill):
        raises(ValueError, f, q[0], k[0], v[0], 4)
        raises(ValueError, f, q, k, v[:, :4], 4)
        raises(ValueError, f, q[:, :4], k, v, 4)
        raises(ValueError, f, q[..., :32], k, v, 4)
        raises(ValueError, f, e(2, 5, 3, 64), k, v, 4)
        raises(ValueError, f, q[:, :0], k[:, :0], v[:, :0], 4)
        raises(ValueError, f, q, k, v, 0)
        raises(ValueError, f, q, k, v, 4, -1)
        raises(ValueError, f, q, k, v, 4, scale=0.0)
        raises(ValueError, f, q, k, v, 4, scale=-1.0)
        raises(ValueError, f, q, k, v, 4, scale=float("nan"))
        raises(ValueError, f, q, k, v, 4, scale=float("inf"))
        raises(ValueError, f, q, k.half(), v, 4)
        raises(NotImplementedError, f, q, k, v, 4, 65)
        raises(NotImplementedError, f, q.float(), k.float(), v.float(), 4)
        raises(NotImplementedError, f, q[..., :60], k[..., :60], v[..., :60], 4)
        raises(NotImplementedError, f, e(1, 2, 1, 136), e(1, 2, 1, 136), e(1, 2, 1, 136), 4)
        raises(RuntimeError, f, q, k, v, 4)


def test_sliding_state_and_step():
    kc, vc, n = e(2, 2, 6, 64), e(2, 2, 6, 64), torch.zeros(2, dtype=torch.int32)
    raises(ValueError, SlidingState, kc, vc, n, 4, 1)
    raises(ValueError, SlidingState, kc, vc[:1], n, 4, 2)
    raises(ValueError, SlidingState, kc, vc.half(), n, 4, 2)
    raises(ValueError, SlidingState, kc, vc, n[:1], 4, 2)
    raises(ValueError, SlidingState, kc, vc, n.long(), 4, 2)
    raises(ValueError, SlidingState, kc.transpose(0, 1), vc.transpose(0, 1), n, 4, 2)
    s = SlidingState(kc, vc, n, 4, 2)
    q, k = e(2, 4, 64), e(2, 2, 64)
    f = sliding_window_step
    raises(ValueError, f, s, q[:, None], k, k)
    raises(ValueError, f, s, q, e(2, 1, 64), e(2, 1, 64))
    raises(ValueError, f, s, q[:1], k[:1], k[:1])
    raises(ValueError, f, s, q.half(), k.half(), k.half())
    raises(ValueError, f, s, q, k, k, scale=0.0)
    raises(RuntimeError, f, s, q, k, k)


# ------------------------------------------------------------------- the C-ABI's codes
P = ctypes.c_void_p
OK, VAL, NOT = _lib.HATTN_OK, _lib.HATTN_ERR_VALUE, _lib.HATTN_ERR_NOT_IMPLEMENTED


def code(name, *args, **want):
    st = getattr(_lib.load(), name)(*args)
    assert st != OK and _lib.load().hattn_last_error()
    return st


@pytest.mark.parametrize("rows,n,dx,dr,dw,st", [
    (0, 16, 0, 0, 0, VAL), (4, 0, 0, 0, 0, VAL), (4, 16385, 0, 0, 0, NOT), (4, 16, 3, 3, 0, NOT),
    (4, 16, 0, 1, 0, NOT), (4, 16, 0, 0, -1, NOT), (4, 16, 0, 0, 0, VAL)])  # the last: null tensors
def test_layer_norm_codes(rows, n, dx, dr, dw, st):
    fake = 16 if st == NOT else None  # placeholders that no launch sees
    assert code("hattn_layer_norm_fwd", None, fake, None, None, None, None, None, None, rows, n,
                1e-5, dx, dr, dw, None) == st
    assert code("hattn_layer_norm_bwd", *([None] * 10), rows, n, dx, dr, dw, None, 0, None) == st


@pytest.mark.parametrize("B,T,D,dx,dg,st", [
    (0, 1, 1, 0, 0, VAL), (1, 0, 1, 0, 0, VAL), (1, 1, 0, 0, 0, VAL), (1, 1, 1, 0, 1, NOT),
    (1, 1, 1, 5, 5, NOT), (1, 2 ** 30 + 1, 1, 2, 2, NOT), (1 << 20, 1 << 20, 64, 0, 0, NOT), (1, 8, 8, 0, 2, VAL)])
def test_recurrence_codes(B, T, D, dx, dg, st):
    assert code("hattn_gated_recurrence_fwd", *([None] * 7), B, T, D, dx, dg, None, 0, None) == st
    assert code("hattn_gated_recurrence_bwd", *([None] * 9), B, T, D, dx, dg, None, 0, None) == st
    if T == 1:
        assert code("hattn_gated_recurrence_step", *([None] * 4), B, D, dx, dg, None) == st


@pytest.mark.parametrize("kw,st", [
    (dict(B=0), VAL), (dict(H=3), VAL), (dict(window=0), VAL), (dict(sinks=-1), VAL),
    (dict(scale=0.0), VAL), (dict(scale=float("nan")), VAL), (dict(sinks=65), NOT),
    (dict(D=60), NOT), (dict(D=136), NOT), (dict(dtype=2), NOT), (dict(H=2 ** 18, G=2 ** 18), NOT),
    (dict(), VAL)])
def test_sliding_codes(kw, st):
    a = dict(B=1, T=4, H=4, G=2, D=64, window=4, sinks=0, scale=0.125, dtype=0)
    a.update(kw)
    dims = [a[n] for n in ("B", "T", "H", "G", "D", "window", "sinks")]
    assert code("hattn_sliding_fwd", *([None] * 7), *dims, a["scale"], a["dtype"], None) == st
    assert code("hattn_sliding_bwd", *([None] * 11), *dims, a["scale"], a["dtype"], None, 0, None) == st
    step = [a[n] for n in ("B", "H", "G", "D", "window", "sinks")]
    assert code("hattn_sliding_step", *([None] * 7), *step, a["scale"], a["dtype"], None, 0, None) == st
    if "H" not in kw and "scale" not in kw:
        fill = [a[n] for n in ("B", "T", "G", "D", "window", "sinks")]
        assert code("hattn_sliding_cache_fill", *([None] * 7), *fill, a["dtype"], None) == st


def test_workspace_queries():
    lib = _lib.load()
    assert lib.hattn_layer_norm_bwd_workspace(4, 16) == 4 * 2 * 16 * 4
    assert lib.hattn_layer_norm_bwd_workspace(100000, 16) == 1024 * 2 * 16 * 4
    assert lib.hattn_layer_norm_bwd_workspace(100000, 4096) == 512 * 2 * 4096 * 4
    assert lib.hattn_layer_norm_bwd_workspace(0, 16) == 0
    # fp32, or an odd number of channels: 256 tokens a segment, strips of 64; else 128 and 128
    assert lib.hattn_gated_recurrence_segments(256, 100, 2) == 1
    assert lib.hattn_gated_recurrence_segments(257, 101, 0) == 2
    assert lib.hattn_gated_recurrence_segments(256, 100, 1) == 2
    assert lib.hattn_gated_recurrence_segments(0, 100, 1) == 0
    assert lib.hattn_gated_recurrence_workspace(2, 256, 100, 2) == 0
    assert lib.hattn_gated_recurrence_workspace(2, 257, 100, 2) == 2 * 2 * 128 * 8
    assert lib.hattn_gated_recurrence_workspace(2, 257, 130, 0) == 3 * 2 * 256 * 8
    assert lib.hattn_gated_recurrence_workspace(0, 257, 100, 2) == 0
    # delta, and the sinks' partial sums: the near one and a (chunk of 1024, head) each
    delta = 2 * 4 * 3000 * 4
    assert lib.hattn_sliding_bwd_workspace(2, 3000, 4, 2, 64, 3000, 8) == delta
    assert lib.hattn_sliding_bwd_workspace(2, 3000, 4, 2, 64, 100, 0) == delta
    assert lib.hattn_sliding_bwd_workspace(2, 3000, 4, 2, 64, 100, 8) == \
        delta + (1 + 3 * 2) * 2 * 2 * 8 * 2 * 64 * 4
    assert lib.hattn_sliding_step_workspace(1, 4, 2, 64, 120, 8) == 4 * 1 * 66 * 4
    assert lib.hattn_sliding_step_workspace(1, 4, 2, 64, 0, 8) == 0
