"""Refusals of the global attention's operators (rotary positions, the cache in 8 bits, attention over
it): the package's exceptions and the C-ABI's status codes, on the host, before any launch; and the
frequencies of longer contexts."""
import ctypes
import math

import pytest
import torch

from hattention import _lib
from hattention.quant_cache_apis import (E4M3, QuantCache, quant_cache_append,
                                         quant_cache_attention, quant_cache_read, quant_cache_step)
from hattention.rotary_apis import rotary_embedding, rotary_frequencies

BF, FH, FS = torch.bfloat16, torch.float16, torch.float32
e = lambda *s, dtype=BF: torch.zeros(*s, dtype=dtype)


def raises(kind, fn, *args, **kw):
    with pytest.raises(kind):
        fn(*args, **kw)


def test_rotary():
    q, k, f = e(2, 5, 4, 64), e(2, 5, 2, 64), torch.ones(16)
    g = rotary_embedding
    raises(ValueError, g, q[0, 0], None, f)
    raises(ValueError, g, q, k[0], f)
    raises(ValueError, g, q, k[:, :4], f)
    raises(ValueError, g, q, k[..., :32], f)
    raises(ValueError, g, q[:, :0], k[:, :0], f)
    raises(ValueError, g, q, k[:, :, :0], f)
    raises(ValueError, g, q, k.half(), f)
    raises(NotImplementedError, g, q.double(), k.double(), f)
    raises(ValueError, g, q, k, torch.ones(33))
    raises(ValueError, g, q, k, torch.ones(0))
    raises(ValueError, g, q, k, torch.ones(4, 4))
    raises(NotImplementedError, g, q, k, f.half())
    raises(NotImplementedError, g, e(1, 1, 1, 514), None, f)
    raises(ValueError, g, q, k, f, layout="pairs")
    raises(ValueError, g, q, k, f, scale=float("nan"))
    raises(ValueError, g, q, k, f, scale=float("inf"))
    i = torch.zeros(2, dtype=torch.int64)
    raises(ValueError, g, q, k, f, i[:1])
    raises(ValueError, g, q, k, f, torch.zeros(2, 4, dtype=torch.int64))
    raises(ValueError, g, q, k, f, torch.zeros((), dtype=torch.int64))
    raises(NotImplementedError, g, q, k, f, i.float())
    raises(ValueError, g, q[:, 0], k[:, 0], f)  # one token a row needs positions
    raises(ValueError, g, q[:, 0], k[:, 0], f, torch.zeros(2, 4, dtype=torch.int64))
    raises(RuntimeError, g, q, k, f, i)         # not on a HIP device


def test_frequencies():
    f = lambda *a, **kw: rotary_frequencies(*a, device="cpu", **kw)
    for dim in (0, 3, -2):
        raises(ValueError, f, dim)
    raises(ValueError, f, 8, 1.0)
    raises(ValueError, f, 8, math.inf)
    raises(ValueError, f, 8, scaling="other")
    raises(ValueError, f, 8, scaling="linear", factor=0.5)
    raises(ValueError, f, 2, scaling="ntk", factor=2.0)
    raises(ValueError, f, 8, scaling="yarn", factor=2.0)
    raises(ValueError, f, 8, scaling="yarn", factor=2.0, original_length=0)
    raises(ValueError, f, 8, scaling="yarn", factor=2.0, original_length=64, fast=1.0)
    plain, scale = f(64)
    assert plain.dtype == torch.float64 and plain.shape == (32,) and scale == 1.0
    assert plain[0] == 1.0
    assert torch.allclose(plain[1:] / plain[:-1], torch.tensor(1e4 ** (-1 / 32), dtype=torch.float64),
                          rtol=1e-14)
    linear, scale = f(64, scaling="linear", factor=4.0)
    assert scale == 1.0 and torch.equal(linear, plain / 4)
    # the fastest stays, the slowest is divided by the factor
    ntk, scale = f(64, scaling="ntk", factor=4.0)
    assert scale == 1.0 and ntk[0] == 1.0
    assert abs(ntk[-1] / (plain[-1] / 4) - 1) < 1e-13
    # turns in 4096 tokens: above 32 they stay, below 1 they are divided, between by the formula
    yarn, scale = f(64, scaling="yarn", factor=4.0, original_length=4096)
    assert scale == 1 + 0.1 * math.log(4)
    turns = 4096 * plain / (2 * math.pi)
    stay = ((turns - 1) / 31).clamp(0, 1)
    assert (stay == 1).any() and (stay == 0).any() and ((stay > 0) & (stay < 1)).any()
    assert torch.equal(yarn[stay == 1], plain[stay == 1])
    assert torch.allclose(yarn[stay == 0], plain[stay == 0] / 4, rtol=1e-15)
    assert torch.allclose(yarn, plain * stay + plain / 4 * (1 - stay), rtol=1e-14)
    same, scale = f(64, scaling="yarn", factor=1.0, original_length=4096)
    assert scale == 1.0 and torch.allclose(same, plain, rtol=1e-15)


def parts(B=2, G=2, slots=128, D=64):
    z = lambda: torch.zeros(B, G, slots, D, dtype=torch.uint8).view(E4M3)
    s = lambda: torch.ones(B, G, slots // 64)
    return [z(), z(), s(), s(), torch.zeros(B, dtype=torch.int32)]


def test_cache():
    ok = parts()
    c = QuantCache(*ok)
    assert c.capacity == 128
    for i, bad in ((0, ok[0][0]), (1, ok[1][:1]), (2, ok[2][:, :, :1]), (3, ok[3][:1]),
                   (4, ok[4][:1])):
        raises(ValueError, QuantCache, *(bad if j == i else t for j, t in enumerate(ok)))
    for i, dtype in ((0, BF), (1, torch.float8_e5m2), (2, BF), (3, torch.float64), (4, torch.int64)):
        raises(ValueError, QuantCache, *(t.to(dtype) if j == i else t for j, t in enumerate(ok)))
    raises(ValueError, QuantCache, *(t[:, :, :100] if j < 2 else t for j, t in enumerate(ok)))
    raises(ValueError, QuantCache, *(t.transpose(0, 1) if j < 4 else t for j, t in enumerate(ok)))
    raises(ValueError, QuantCache, *(t[:0] for t in ok))
    raises(NotImplementedError, QuantCache, *parts(D=24))
    raises(NotImplementedError, QuantCache, *parts(D=144))
    flat = torch.zeros(2 * 2 * 128 * 64 + 8, dtype=torch.uint8)[8:].view(E4M3).view(2, 2, 128, 64)
    if flat.data_ptr() % 16:
        raises(ValueError, QuantCache, flat, *ok[1:])
    raises(ValueError, QuantCache.empty, 1, 1, 64, 0, device="cpu")
    raises(ValueError, QuantCache.empty, 0, 1, 64, 64, device="cpu")
    c = QuantCache.empty(3, 2, 48, 65, device="cpu")
    assert c.k.shape == (3, 2, 128, 48) and c.k_scale.shape == (3, 2, 2)
    assert not c.counts.any() and not c.k.float().any() and (c.v_scale == 1).all()


def test_append_and_read():
    c = QuantCache(*parts())
    k = e(2, 5, 2, 64)
    f = quant_cache_append
    raises(ValueError, f, c, k[0], k[0])
    raises(ValueError, f, c, k[:, :0], k[:, :0])
    raises(ValueError, f, c, k, k[:, :4])
    raises(ValueError, f, c, k[:1], k[:1])
    raises(ValueError, f, c, e(2, 5, 4, 64), e(2, 5, 4, 64))
    raises(ValueError, f, c, k[..., :48], k[..., :48])
    raises(ValueError, f, c, k, k.half())
    raises(NotImplementedError, f, c, k.float(), k.float())
    raises(ValueError, f, c, e(2, 129, 2, 64), e(2, 129, 2, 64))
    raises(RuntimeError, f, c, k, k)
    f = quant_cache_read
    for lo, hi in ((-1, 4), (4, 4), (5, 4), (0, 129), (128, None)):
        raises(ValueError, f, c, BF, lo, hi)
    raises(NotImplementedError, f, c, torch.float64)
    raises(RuntimeError, f, c)


def test_attention_and_step():
    c = QuantCache(*parts())
    q, k = e(2, 5, 4, 64), e(2, 2, 64)
    f = quant_cache_attention
    raises(ValueError, f, c, q[0])
    raises(ValueError, f, c, q[:1])
    raises(ValueError, f, c, q[..., :48])
    raises(ValueError, f, c, q[:, :, :3])
    raises(ValueError, f, c, q[:, :0])
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        raises(ValueError, f, c, q, scale)
    raises(NotImplementedError, f, c, q.float())
    raises(RuntimeError, f, c, q)
    f = quant_cache_step
    raises(ValueError, f, c, q, k, k)
    raises(ValueError, f, c, q[:, 0], q[:, 0], q[:, 0])
    raises(ValueError, f, c, q[:, 0], k, k[:1])
    raises(ValueError, f, c, q[:, 0], k[:, None], k[:, None])
    raises(ValueError, f, c, q[:, 0], k.half(), k.half())
    raises(ValueError, f, c, q[:, 0], k, k, 0.0)
    raises(NotImplementedError, f, c, q[:, 0].float(), k.float(), k.float())
    raises(RuntimeError, f, c, q[:, 0], k, k)


# ------------------------------------------------------------------- the C-ABI's codes
OK, VAL, NOT = _lib.HATTN_OK, _lib.HATTN_ERR_VALUE, _lib.HATTN_ERR_NOT_IMPLEMENTED


def code(name, *args):
    st = getattr(_lib.load(), name)(*args)
    assert st != OK and _lib.load().hattn_last_error()
    return st


@pytest.mark.parametrize("kw,st", [
    (dict(B=0), VAL), (dict(T=0), VAL), (dict(H=0), VAL), (dict(G=-1), VAL), (dict(pairs=0), VAL),
    (dict(pairs=33), VAL), (dict(scale=float("nan")), VAL), (dict(scale=float("inf")), VAL),
    (dict(dtype=3), NOT), (dict(D=514), NOT), (dict(H=2 ** 20 + 1), NOT),
    (dict(B=2 ** 20, T=2 ** 20), NOT), (dict(), VAL)])  # the last: null tensors
def test_rotary_codes(kw, st):
    a = dict(B=1, T=4, H=4, G=2, D=64, pairs=32, scale=1.0, dtype=0)
    a.update(kw)
    p = 16 if st == NOT else None  # placeholders that no launch sees
    strides = (ctypes.c_longlong * 6)(0, 0, 0, 0, 0, 0)
    assert code("hattn_rotary", p, p, strides, p, p, p, 1, None, 0, 0, 0, 0,
                *(a[n] for n in ("B", "T", "H", "G", "D", "pairs")), 0, a["scale"], 0, a["dtype"],
                None) == st


@pytest.mark.parametrize("kw,st", [
    (dict(B=0), VAL), (dict(G=0), VAL), (dict(D=0), VAL), (dict(capacity=0), VAL),
    (dict(capacity=100), VAL), (dict(T=0, H=4), VAL), (dict(D=24), NOT), (dict(D=144), NOT),
    (dict(capacity=2 ** 30 + 64), NOT), (dict(B=2 ** 16, G=2 ** 16, H=2 ** 16), NOT),
    (dict(dtype=2), NOT), (dict(), VAL)])
def test_cache_codes(kw, st):
    a = dict(B=1, T=4, H=4, G=2, D=64, capacity=128, scale=0.125, dtype=0)
    a.update(kw)
    new = [a[n] for n in ("B", "T", "G", "D", "capacity", "dtype")]
    assert code("hattn_quant_cache_append", *([None] * 9), *new, None) == st
    if "dtype" not in kw and "T" not in kw:
        old = [a[n] for n in ("B", "G", "D", "capacity")]
        assert code("hattn_quant_cache_read", *([None] * 7), *old, 0, 4, 0, None) == st
    dims = [a[n] for n in ("B", "T", "H", "G", "D", "capacity")]
    assert code("hattn_quant_cache_attention", *([None] * 9), *dims, a["scale"], a["dtype"], None, 0,
                None) == st
    if "T" not in kw:
        step = [a[n] for n in ("B", "H", "G", "D", "capacity")]
        assert code("hattn_quant_cache_step", *([None] * 10), *step, a["scale"], a["dtype"], None, 0,
                    None) == st


def test_more_codes():
    assert code("hattn_quant_cache_append", *([None] * 9), 1, 129, 2, 64, 128, 0, None) == VAL
    for start, n in ((0, 0), (-1, 4), (125, 4), (0, 129), (2 ** 31 - 1, 2 ** 31 - 1)):
        assert code("hattn_quant_cache_read", *([None] * 7), 1, 2, 64, 128, start, n, 0, None) == VAL
    assert code("hattn_quant_cache_read", *([None] * 7), 1, 2, 64, 128, 0, 4, 3, None) == NOT
    att = lambda *dims: code("hattn_quant_cache_attention", *([None] * 9), *dims, 0, None, 0, None)
    assert att(1, 4, 3, 2, 64, 128, 1.0) == VAL
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert att(1, 4, 4, 2, 64, 128, scale) == VAL
    assert att(1, 2 ** 30, 64, 2, 64, 128, 1.0) == NOT
    assert att(2 ** 13, 2 ** 13, 32, 1, 64, 128, 1.0) == NOT
    # a long prompt's queries are more than a join takes, which it does not need
    assert att(1, 2 ** 18, 64, 8, 64, 2 ** 18, 1.0) == VAL


@pytest.mark.skipif(torch.cuda.is_available(), reason="passes placeholder device pointers")
def test_alignment_strides_and_workspace_codes():
    p, s = 64, lambda *x: (ctypes.c_longlong * len(x))(*x)
    dims = 1, 4, 4, 2, 64, 128
    att = lambda q, st, ws, n: code("hattn_quant_cache_attention", q, None, st, p, p, p, p, p, p,
                                    *dims, 1.0, 0, ws, n, None)
    good = s(1024, 256, 64)
    need = _lib.load().hattn_quant_cache_attention_workspace(*dims)
    assert need == 4 * 4 * 1 * 66 * 4 + 4
    assert att(72, good, p, need) == VAL
    assert att(p, s(1024, 252, 64), p, need) == VAL
    assert att(p, s(1024, -256, 64), p, need) == VAL
    assert att(p, good, None, need) == VAL
    assert att(p, good, p, need - 1) == VAL
    assert att(p, good, p + 8, need) == VAL
    assert code("hattn_quant_cache_append", p, p, None, s(64, 64, 60, 64, 64, 64), p, p, p, p, p, 1, 4,
                2, 64, 128, 0, None) == VAL
    assert code("hattn_quant_cache_append", p, 72, None, s(64, 64, 64, 64, 64, 64), p, p, p, p, p, 1, 4,
                2, 64, 128, 0, None) == VAL
    assert code("hattn_rotary", 65, None, s(0, 0, 0, 0, 0, 0), p, None, p, 1, None, 0, 0, 0, 0, 1, 1, 1,
                0, 64, 32, 0, 1.0, 0, 0, None) == VAL
    assert code("hattn_rotary", p, None, s(0, 0, 0, 0, 0, 0), p, None, 68, 1, None, 0, 0, 0, 0, 1, 1, 1,
                0, 64, 32, 0, 1.0, 0, 0, None) == VAL


def test_workspace_query():
    f = _lib.load().hattn_quant_cache_attention_workspace
    # few queries: parts of at least 256 tokens, at most 256 of them, as many as fill the card
    assert f(1, 1, 4, 4, 64, 256) == 4 * 1 * 66 * 4 + 4
    assert f(1, 1, 4, 4, 64, 64 * 1024) == 4 * 256 * 66 * 4 + 4
    assert f(0, 1, 4, 4, 64, 256) == 0
    assert f(1, 1, 4, 4, 60, 256) == 0
