"""The cache in 8 bits: codes and scales bit for bit against the definition in 64 bits, whatever
calls the tokens came in."""
import math

import pytest
import torch

from hattention.quant_cache_apis import BLOCK, E4M3, QuantCache, quant_cache_append, quant_cache_read, \
    quant_cache_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FH, FS = torch.bfloat16, torch.float16, torch.float32
MOST = {BF: 119, FH: 7}


def make(seed, *shape, dtype=BF, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * scale).to(dtype).to(DEV)


def e4m3(y):
    """The nearest code's value, ties to even; NaN for what is not finite."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6)) + 1e-9) - 3)
    return (torch.round(y / step) * step).clamp(-448, 448).masked_fill(~y.isfinite(), math.nan)


def exponent(y, dtype):
    top = y.abs().masked_fill(~y.isfinite(), 0).max()
    e = -100 if top == 0 else math.ceil(math.log2(top / 448) - 1e-9)
    return min(max(e, -100), MOST[dtype])


class Oracle:
    """One of k and v: codes' values and scales on the CPU in 64 bits, row by row."""

    def __init__(self, B, G, slots, D):
        self.codes = torch.zeros(B, G, slots, D, dtype=torch.float64)
        self.scale = torch.ones(B, G, slots // BLOCK, dtype=torch.float64)

    def append(self, b, n, x, dtype):
        """Tokens x [t, G, D] after the n of row b."""
        x = x.double().cpu()
        at, end = n, min(n + x.shape[0], self.codes.shape[2])
        while at < end:
            j, top = at // BLOCK, min((at // BLOCK + 1) * BLOCK, end)
            for g in range(x.shape[1]):
                y = x[at - n:top - n, g]
                s = 2.0 ** exponent(y, dtype)
                if at > j * BLOCK:
                    was = float(self.scale[b, g, j])
                    s = max(s, was)
                    old = self.codes[b, g, j * BLOCK:at]
                    old.copy_(e4m3(old * (was / s)))
                self.codes[b, g, at:top] = e4m3(y / s)
                self.scale[b, g, j] = s
            at = top


def fresh(B, G, slots, D):
    """A cache whose slots and scales are NaN until they are written."""
    k, v = (torch.full((B, G, slots, D), 0x7f, dtype=torch.uint8, device=DEV).view(E4M3)
            for _ in range(2))
    ks, vs = (torch.full((B, G, slots // BLOCK), math.nan, device=DEV) for _ in range(2))
    return QuantCache(k, v, ks, vs, torch.zeros(B, dtype=torch.int32, device=DEV))


def same(cache, k, v, counts):
    assert cache.counts.tolist() == counts
    for codes, scale, want in ((cache.k, cache.k_scale, k), (cache.v, cache.v_scale, v)):
        codes, scale = codes.float().double().cpu(), scale.double().cpu()
        for b, n in enumerate(counts):
            n = min(n, codes.shape[2])
            blocks = -(-n // BLOCK)
            assert torch.equal(scale[b, :, :blocks], want.scale[b, :, :blocks])
            assert torch.equal(codes[b, :, :n].nan_to_num(999), want.codes[b, :, :n].nan_to_num(999))
            # nothing behind a row's tokens was touched
            assert codes[b, :, n:].isnan().all() and scale[b, :, blocks:].isnan().all()


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("G,D", [(1, 16), (2, 32), (1, 48), (3, 64), (2, 80), (1, 96), (1, 112), (2, 128)])
def test_append_in_pieces(dtype, G, D):
    B, slots = 3, 320
    cache, ok, ov = fresh(B, G, slots, D), Oracle(B, G, slots, D), Oracle(B, G, slots, D)
    n = [0] * B
    for i, (T, lens) in enumerate([(1, None), (7, [7, 0, 3]), (62, None), (130, [130, 64, 1]),
                                   (1, [1, 1, 0]), (64, [2, 64, 33])]):
        # pieces grow and shrink, so that scales do too
        size = [1.0, 0.01, 30.0, 1e-4, 700.0, 3.0][i]
        k, v = make(10 + i, B, T, G, D, dtype=dtype, scale=size), \
            make(20 + i, B, T, G, D, dtype=dtype, scale=1 / size)
        lengths = None if lens is None else torch.tensor(lens, device=DEV)
        assert quant_cache_append(cache, k, v, lengths) is cache
        for b in range(B):
            t = T if lens is None else lens[b]
            ok.append(b, n[b], k[b, :t], dtype)
            ov.append(b, n[b], v[b, :t], dtype)
            n[b] += t
        same(cache, ok, ov, n)


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("G,D", [(1, 16), (9, 64), (2, 128), (3, 80)])
def test_step_appends_as_append_does(dtype, G, D):
    B = 3
    a, b = fresh(B, G, 192, D), fresh(B, G, 192, D)
    ok, ov = Oracle(B, G, 192, D), Oracle(B, G, 192, D)
    k, v = make(1, B, 60, G, D, dtype=dtype, scale=0.1), make(2, B, 60, G, D, dtype=dtype)
    start = [60, 0, 33]
    for c in (a, b):
        quant_cache_append(c, k, v, torch.tensor(start, device=DEV))
    for i in range(3):
        ok.append(i, 0, k[i, :start[i]], dtype)
        ov.append(i, 0, v[i, :start[i]], dtype)
    for i in range(8):
        k, v = (make(30 + 2 * i + j, B, G, D, dtype=dtype, scale=2.0 ** (i - 3)) for j in range(2))
        quant_cache_append(a, k[:, None], v[:, None])
        quant_cache_step(b, make(50 + i, B, G, D, dtype=dtype), k, v)
        for r in range(B):
            ok.append(r, start[r] + i, k[r][None], dtype)
            ov.append(r, start[r] + i, v[r][None], dtype)
        for c in (a, b):
            same(c, ok, ov, [n + i + 1 for n in start])


@pytest.mark.parametrize("dtype", [BF, FH])
def test_every_value(dtype):
    """All 16-bit patterns, in blocks whose largest value is each of several, ties among them."""
    x = torch.arange(2 ** 16, dtype=torch.int32).to(torch.int16).view(dtype)
    x = x[x.isfinite()]
    x = x[torch.argsort(x.float().abs(), stable=True)]  # a block's values are near each other
    T = x.numel() // 16 // 64 * 64
    tops = x[:T * 16].view(1, T, 1, 16).to(DEV)
    mixed = tops.flatten()[torch.randperm(T * 16, generator=torch.Generator().manual_seed(1)).to(DEV)]
    for k, v in ((tops, mixed.view(1, T, 1, 16)),):
        cache, ok, ov = fresh(1, 1, T, 16), Oracle(1, 1, T, 16), Oracle(1, 1, T, 16)
        quant_cache_append(cache, k, v)
        ok.append(0, 0, k[0], dtype)
        ov.append(0, 0, v[0], dtype)
        same(cache, ok, ov, [T])
        got = quant_cache_read(cache, FS)
        assert got[0].isfinite().all() and got[1].isfinite().all()
        # a value's one rounding
        err = (got[0] - k.float()).abs().view(T // 64, -1)
        scale = cache.k_scale[0, 0][:, None]
        bound = torch.maximum(k.float().abs().view(T // 64, -1) * 2.0 ** -4, scale * 2.0 ** -10)
        fits = k.float().abs().view(T // 64, -1) <= 448 * scale
        assert (fits.all(1) | (scale[:, 0] == 2.0 ** MOST[dtype])).all()
        assert (err <= bound)[fits].all()


@pytest.mark.parametrize("dtype", [BF, FH])
def test_what_is_not_finite(dtype):
    k = make(1, 1, 70, 2, 32, dtype=dtype)
    v = make(2, 1, 70, 2, 32, dtype=dtype)
    k[0, 3, 0, 5], k[0, 66, 1, 0], k[0, 9, 1, 31] = math.inf, math.nan, -math.inf
    v[0, 64:] = math.nan  # a whole block
    cache, ok, ov = fresh(1, 2, 128, 32), Oracle(1, 2, 128, 32), Oracle(1, 2, 128, 32)
    quant_cache_append(cache, k, v)
    ok.append(0, 0, k[0], dtype)
    ov.append(0, 0, v[0], dtype)
    same(cache, ok, ov, [70])
    # it stays NaN where the scale grows, and a later call is not touched by it
    more = make(3, 1, 20, 2, 32, dtype=dtype, scale=50.0)
    quant_cache_append(cache, more, more)
    ok.append(0, 70, more[0], dtype)
    ov.append(0, 70, more[0], dtype)
    same(cache, ok, ov, [90])
    got = quant_cache_read(cache, BF, 0, 90)
    assert torch.equal(got[0][:, :70].isnan(), ~k.isfinite())


def test_zeros_and_growth_from_them():
    cache, ok = fresh(1, 1, 64, 16), Oracle(1, 1, 64, 16)
    z = torch.zeros(1, 5, 1, 16, dtype=BF, device=DEV)
    quant_cache_append(cache, z, z)
    ok.append(0, 0, z[0], BF)
    same(cache, ok, ok, [5])
    x = make(1, 1, 5, 1, 16)
    quant_cache_append(cache, x, x)
    ok.append(0, 5, x[0], BF)
    same(cache, ok, ok, [10])


def test_capacity():
    """Tokens past it are counted and not stored; a count set back takes the row into use again."""
    B, G, D = 2, 2, 32
    cache, ok, ov = fresh(B, G, 128, D), Oracle(B, G, 128, D), Oracle(B, G, 128, D)
    k, v = make(1, B, 100, G, D), make(2, B, 100, G, D)
    n = [0, 0]
    for lens in ([100, 20], [100, 100], [100, 100], [100, 100]):
        quant_cache_append(cache, k, v, torch.tensor(lens, device=DEV))
        for b in range(B):
            if n[b] < 128:
                ok.append(b, n[b], k[b, :lens[b]], BF)
                ov.append(b, n[b], v[b, :lens[b]], BF)
            n[b] += lens[b]
        same(cache, ok, ov, n)
    quant_cache_step(cache, make(3, B, G, D), k[:, 0], v[:, 0])
    n = [m + 1 for m in n]
    same(cache, ok, ov, n)
    cache.counts.fill_(2 ** 31 - 2)
    for _ in range(3):
        quant_cache_append(cache, k, v)
        quant_cache_step(cache, make(3, B, G, D), k[:, 0], v[:, 0])
    assert cache.counts.tolist() == [2 ** 31 - 1] * B
    # back into the middle of a block, whose scale stays, and to the start, whose scale is made again
    cache.counts.copy_(torch.tensor([70, 0]))
    again = make(4, B, 3, G, D, scale=0.01)
    quant_cache_append(cache, again, again)
    for b, at in ((0, 70), (1, 0)):
        ok.append(b, at, again[b], BF)
        ov.append(b, at, again[b], BF)
    for codes, scale, want in ((cache.k, cache.k_scale, ok), (cache.v, cache.v_scale, ov)):
        assert torch.equal(codes.float().double().cpu()[0, :, :73], want.codes[0, :, :73])
        assert torch.equal(codes.float().double().cpu()[1, :, :3], want.codes[1, :, :3])
        assert torch.equal(scale.double().cpu()[:, :, 0], want.scale[:, :, 0])
    cache.counts.fill_(-5)  # taken as 0
    quant_cache_append(cache, again, again, torch.tensor([2, -7], device=DEV))
    assert cache.counts.tolist() == [2, 0]


def test_views_and_lengths():
    B, T, G, D = 2, 21, 2, 64
    wide = make(1, B, T, 6 * D)
    pairs = [tuple(t.unflatten(-1, (G, D)) for t in wide.split(2 * D, -1)[:2]),
             tuple(make(2 + i, B, G, T, D).transpose(1, 2) for i in range(2)),
             tuple(make(4 + i, B, T, G, D + 3)[..., 3:] for i in range(2)),
             tuple(make(6 + i, 1, 1, 1, D).expand(B, T, G, D) for i in range(2)),
             tuple(make(8 + i, 2 * B, 2 * T, G, D)[::2, ::2] for i in range(2))]
    for k, v in pairs:
        want, got = fresh(B, G, 64, D), fresh(B, G, 64, D)
        quant_cache_append(want, k.contiguous(), v.contiguous(), torch.tensor([21, 5], device=DEV))
        n = torch.tensor([2 ** 40, 5], device=DEV)  # clamped to T
        x = k.clone(memory_format=torch.preserve_format)
        quant_cache_append(got, k, v, n)
        assert torch.equal(x, k)
        for a, b in zip(want._tensors(), got._tensors()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        a, b = fresh(B, G, 64, D), fresh(B, G, 64, D)
        quant_cache_step(a, k[:, 0], k[:, 0], v[:, 0])
        quant_cache_step(b, k[:, 0].contiguous(), k[:, 0].contiguous(), v[:, 0].contiguous())
        for x, y in zip(a._tensors(), b._tensors()):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("dtype", [BF, FH, FS])
@pytest.mark.parametrize("G,D", [(1, 16), (3, 32), (2, 64), (2, 80), (1, 128)])
def test_read(dtype, G, D):
    B, slots = 3, 256
    cache = fresh(B, G, slots, D)
    k, v = make(1, B, 200, G, D, scale=3.0), make(2, B, 200, G, D, scale=0.2)
    lens = [200, 0, 67]
    quant_cache_append(cache, k, v, torch.tensor(lens, device=DEV))
    val = [(c.float().view(B, G, -1, BLOCK, D) * s[..., None, None]).view(B, G, slots, D).transpose(1, 2)
           for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]
    held = (torch.arange(slots, device=DEV) < cache.counts[:, None])[..., None, None]
    for start, stop in ((0, None), (0, 1), (63, 65), (64, 128), (66, 200), (199, 256), (255, 256),
                        (5, 64)):
        got = quant_cache_read(cache, dtype, start, stop)
        for x, y in zip(got, val):
            want = torch.where(held, y, 0).to(dtype)[:, start:stop]
            assert x.dtype == dtype and x.is_contiguous() and torch.equal(x, want)


def test_offsets_past_32_bits():
    """A cache of 2.2 G codes: its last row and head, and its first."""
    B, G, D = 2, 4, 128
    slots = 2 ** 21 + 64 * 1000
    cache = QuantCache.empty(B, G, D, slots, device=DEV)
    assert cache.k.numel() > 2 ** 31
    k, v = make(1, B, 100, G, D), make(2, B, 100, G, D)
    cache.counts.copy_(torch.tensor([slots - 64 - 70, 3]))
    cache.counts[1] = slots - 64 - 40
    quant_cache_append(cache, k, v)
    small, ok, ov = QuantCache.empty(B, G, D, 256, device=DEV), Oracle(B, G, 256, D), Oracle(B, G, 256, D)
    lead = [64 - 6, 64 - 40]  # the same places in a block
    for b in range(B):
        ok.append(b, lead[b], k[b], BF)
        ov.append(b, lead[b], v[b], BF)
    got = quant_cache_read(cache, FS, slots - 200, slots)
    for x, codes in zip(got, (ok, ov)):
        val = (codes.codes.view(B, G, -1, BLOCK, D) * codes.scale[..., None, None]).view(B, G, -1, D)
        for b, first in enumerate((slots - 64 - 70, slots - 64 - 40)):
            at = first - (slots - 200)
            want = val[b, :, lead[b]:lead[b] + 100].transpose(0, 1)
            assert torch.equal(x[b, at:at + 100].double().cpu(), want)
    assert not cache.k[0, :, :64].float().any() and not cache.v[1, 0, :1000].float().any()
    del small
