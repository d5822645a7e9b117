"""Attention over the cache in 8 bits against the formula in 64 bits on the cache's own values.

Tolerances count roundings.  With h the half step of q's dtype and u = 2^-24: a probability is
rounded to that dtype and carries the errors of its score (D products in fp32, the block's scale
and the exponent's sum) and of the sum of n: r = h + 2 (D + 8) u max|s| + n u; o = P V errs by
r sum P |v|, then by its own half step.
"""
import math

import pytest
import torch

from hattention.quant_cache_apis import (BLOCK, E4M3, QuantCache, quant_cache_append,
                                         quant_cache_attention, quant_cache_read, quant_cache_step)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
BF, FH, FS = torch.bfloat16, torch.float16, torch.float32


def make(seed, *shape, dtype=BF, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * scale).to(dtype).to(DEV)


def filled(seed, B, G, slots, D, counts, spread=1.0):
    """A cache whose written codes are of every size and whose scales differ from block to block;
    what no token has reached is NaN."""
    gen = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        x = torch.randn(B, G, slots // BLOCK, BLOCK, D, generator=gen)
        s = torch.exp2(torch.randint(-9, -5, (B, G, slots // BLOCK), generator=gen).float() * spread)
        codes = (x / x.abs().amax((-1, -2), keepdim=True) * 448).to(E4M3).view(B, G, slots, D)
        for b, n in enumerate(counts):
            codes.view(torch.uint8)[b, :, n:] = 0x7f
            s[b, :, -(-n // BLOCK):] = math.nan
        out += [codes.to(DEV), s.to(DEV)]
    k, ks, v, vs = out
    return QuantCache(k, v, ks, vs, torch.tensor(counts, dtype=torch.int32, device=DEV))


def values(codes, scale, b, g, n):
    s = scale[b, g].double().repeat_interleave(BLOCK)[:n, None]
    return codes[b, g, :n].float().double() * s


def oracle(cache, q, counts, lens, scale=None):
    """(o, bound) of queries q [B, T, H, D], the last lens[b] tokens of counts[b]."""
    B, T, H, D = q.shape
    G = cache.k.shape[1]
    h = torch.finfo(q.dtype).eps / 2
    scale = D ** -0.5 if scale is None else scale
    o, tol = (torch.zeros(q.shape, dtype=torch.float64, device=DEV) for _ in range(2))
    for b, (n, m) in enumerate(zip(counts, lens)):
        for i in range(H if m and n else 0):
            k, v = (values(c, s, b, i // (H // G), n) for c, s in
                    ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
            x = q[b, :m, i].double()
            hidden = torch.arange(n, device=DEV) > (n - m + torch.arange(m, device=DEV))[:, None]
            p = torch.softmax((x @ k.T * scale).masked_fill(hidden, -math.inf), 1).nan_to_num(0)
            big = (x.abs() @ k.T.abs() * scale).masked_fill(hidden, 0).amax()
            r = h + 2 * (D + 8) * U * big + n * U
            o[b, :m, i] = p @ v
            tol[b, :m, i] = r * (p @ v.abs())
    return o, tol


def close(got, want, tol):
    f = torch.finfo(got.dtype)
    tol = tol + f.eps / 2 * (want.abs() + tol) + f.smallest_normal * f.eps
    over = (got.double() - want).abs() - tol
    assert got.isfinite().all() and not (over > 0).any(), float(over.max())


SIZES = [  # B, T, H, G, D, counts, lengths
    (1, 1, 1, 1, 16, [1], None),
    (1, 1, 4, 4, 64, [2], None),
    (2, 1, 8, 2, 64, [700, 64], None),
    (3, 1, 16, 1, 128, [65, 1000, 4], [1, 1, 0]),
    (2, 1, 40, 2, 80, [513, 255], None),           # 20 queries of a key head
    (2, 1, 33, 1, 128, [300, 129], None),          # 33, two blocks of 32
    (2, 5, 8, 2, 64, [900, 6], [5, 3]),
    (2, 4, 4, 1, 96, [4, 2], None),                # fewer tokens than queries: some see nothing
    (1, 8, 4, 1, 128, [64], None),                 # 32
    (1, 9, 4, 1, 128, [64], None),                 # 36
    (2, 37, 4, 2, 48, [37, 200], [37, 20]),
    (1, 300, 6, 2, 64, [300], None),               # a prompt
    (3, 129, 2, 1, 128, [129, 700, 40], [129, 1, 0]),
    (2, 70, 3, 3, 112, [1000, 70], [70, 70]),
    (2, 16, 4, 1, 128, [200, 64], None),           # 64
    (2, 13, 5, 1, 64, [200, 64], [13, 2]),         # 65
    (1, 64, 16, 1, 128, [3000], None),
    (4, 33, 8, 8, 32, [33, 64, 65, 500], [33, 32, 1, 17]),
]


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("B,T,H,G,D,counts,lens", SIZES)
def test_attention(dtype, B, T, H, G, D, counts, lens):
    slots = -(-max(counts) // BLOCK) * BLOCK
    q = make(1, B, T, H, D, dtype=dtype)
    new = [T] * B if lens is None else lens
    lengths = None if lens is None else torch.tensor(lens, device=DEV, dtype=torch.int32)
    for b, m in enumerate(new):
        q[b, m:] = math.nan  # padding is not used
    # the capacity decides how a row is cut: as it is, and far larger than what is held
    for extra in (0, 64 * BLOCK):
        cache = filled(2, B, G, slots + extra, D, counts)
        o = quant_cache_attention(cache, q, lengths=lengths)
        close(o, *oracle(cache, q, counts, new))
        assert cache.counts.tolist() == counts
        again = quant_cache_attention(cache, q, lengths=lengths)
        assert torch.equal(o, again)


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("T", [1, 40])
def test_long(dtype, T):
    cache = filled(3, 1, 2, 40000 // BLOCK * BLOCK, 64, [39000])
    q = make(4, 1, T, 8, 64, dtype=dtype, scale=2.0)
    close(quant_cache_attention(cache, q, 0.2), *oracle(cache, q, [39000], [T], 0.2))


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("T", [1, 64])
def test_scales_far_apart(dtype, T):
    """Blocks whose scales differ by 2^27 and more, the tokens of the small ones seen too."""
    cache = filled(5, 1, 1, 512, 64, [500], spread=9.0)
    top = 2.0 ** 8 / 448  # the values stay in fp16's range
    cache.v_scale.mul_(2.0 ** 40 * top).clamp_max_(2.0 ** 7)
    cache.k_scale.mul_(2.0 ** 30)
    q = make(6, 1, T, 2, 64, dtype=dtype, scale=0.05)
    q[:, :, 1] = 0  # every token alike
    close(quant_cache_attention(cache, q, 0.01), *oracle(cache, q, [500], [T], 0.01))


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("T", [1, 160])
def test_many_tokens_of_little_weight(dtype, T):
    """One token of weight 1 and 60000 of 2^-24 each, whose values are 2^7 times as large: their part
    of the sum is lost where such weights are rounded to subnormal numbers."""
    n, D = 60000, 64
    slots = -(-n // BLOCK) * BLOCK
    k = torch.zeros(1, 1, slots, D, device=DEV)
    v = torch.full((1, 1, slots, D), 448.0, device=DEV)
    k[0, 0, 5, 0] = 1.0
    v[0, 0, 5] = 3.5
    one = torch.ones(1, 1, slots // BLOCK, device=DEV)
    cache = QuantCache(k.to(E4M3), v.to(E4M3), one, one.clone(),
                       torch.tensor([n], dtype=torch.int32, device=DEV))
    q = torch.zeros(1, T, 1, D, dtype=dtype, device=DEV)
    q[..., 0] = 24.6
    o = quant_cache_attention(cache, q, math.log(2))
    close(o, *oracle(cache, q, [n], [T], math.log(2)))


@pytest.mark.parametrize("T", [1, 64])
def test_large_scores(T):
    """Scores of thousands, of both signs: one token takes all, which need not be the last seen."""
    cache = filled(7, 1, 1, 256, 64, [256])
    q = make(8, 1, T, 4, 64, scale=100.0)
    o = quant_cache_attention(cache, q, 1.0)
    want, tol = oracle(cache, q, [256], [T], 1.0)
    close(o, want, tol)
    # all scores far below zero: queries against the keys they are farthest from
    cache.k.copy_(cache.k.float().abs().to(E4M3))
    q = -q.abs()
    close(quant_cache_attention(cache, q, 1.0), *oracle(cache, q, [256], [T], 1.0))


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("B,H,G,D,start", [
    (1, 1, 1, 16, [0]), (3, 8, 2, 64, [0, 63, 640]), (2, 16, 16, 128, [127, 5]), (2, 34, 2, 80, [300, 64]),
    (5, 6, 1, 112, [1, 2, 3, 4, 1000]), (2, 17, 1, 64, [64, 0]), (1, 66, 2, 128, [700]),
    (2, 130, 1, 64, [90, 1])])
def test_step(dtype, B, H, G, D, start):
    """Each step as append and attention, bit for bit, and near the formula."""
    a = filled(9, B, G, 1088, D, start)
    b = QuantCache(*(t.clone() for t in a._tensors()))
    for i in range(4):
        q, k, v = (make(20 + 3 * i + j, B, n, D, dtype=dtype) for j, n in enumerate((H, G, G)))
        o, same = quant_cache_step(a, q, k, v)
        assert same is a and o.shape == q.shape
        quant_cache_append(b, k[:, None], v[:, None])
        assert torch.equal(o, quant_cache_attention(b, q[:, None])[:, 0])
        for x, y in zip(a._tensors(), b._tensors()):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
        n = [s + i + 1 for s in start]
        close(o[:, None], *oracle(a, q[:, None], n, [1] * B))


@pytest.mark.parametrize("H", [4, 20, 40])
def test_full_and_empty_rows(H):
    """A row past its capacity gives NaN until its count is set back, an empty one zeros."""
    B, G, D = 3, 1, 32
    cache = filled(10, B, G, 64, D, [64, 64, 64])
    for T in (1, 3, 40):
        q = make(11, B, T, H, D)
        cache.counts.copy_(torch.tensor([64, 65, 0]))
        o = quant_cache_attention(cache, q)
        assert o[0].isfinite().all() and o[1].isnan().all() and not o[2].any()
        o = quant_cache_attention(cache, q, lengths=torch.tensor([T, T // 2, T], device=DEV))
        assert o[1, :T // 2].isnan().all() and not o[1, T // 2:].any()
        cache.counts.copy_(torch.tensor([-1, 2 ** 31 - 1, 2]))
        o = quant_cache_attention(cache, q)
        assert not o[0].any() and o[1].isnan().all() and not o[2, :max(T - 2, 0)].any()
        assert o[2, -1].any()
    q, k = make(12, B, H, D), make(13, B, G, D)
    cache.counts.copy_(torch.tensor([63, 64, 70]))
    o, _ = quant_cache_step(cache, q, k, k)
    assert o[0].isfinite().all() and o[1:].isnan().all() and cache.counts.tolist() == [64, 65, 71]
    cache.counts.copy_(torch.tensor([10, 20, 30]))
    o, _ = quant_cache_step(cache, q, k, k)
    close(o[:, None], *oracle(cache, q[:, None], [11, 21, 31], [1] * B))


def test_what_is_not_finite():
    """NaN in k or v of the last token reaches the last query."""
    for T in (2, 80):
        cache = filled(14, 1, 1, 256, 64, [256])
        q = make(15, 1, T, 2, 64)
        clean = quant_cache_attention(cache, q)
        cache.v.view(torch.uint8)[0, 0, 255, 7] = 0x7f  # the last token
        o = quant_cache_attention(cache, q)
        assert o[0, -1, :, 7].isnan().all() and o[0, -1, :, 8:].isfinite().all()
        early = T - 64  # queries whose last token lies in an earlier block
        if early > 0:
            assert torch.equal(o[:, :early], clean[:, :early])
        cache.k.view(torch.uint8)[0, 0, 255, 0] = 0x7f
        o = quant_cache_attention(cache, q)
        assert o[0, -1].isnan().all()
        if early > 0:
            assert torch.equal(o[:, :early], clean[:, :early])
        # a query's own NaN stays its own
        cache = filled(14, 1, 1, 256, 64, [256])
        q[0, 0, 1, 3] = math.nan
        o = quant_cache_attention(cache, q)
        assert o[0, 0, 1].isnan().all() and torch.equal(o[0, 1:], clean[0, 1:])
        assert torch.equal(o[0, 0, 0], clean[0, 0, 0])


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("T,R", [(40, 2), (80, 2), (70, 5), (300, 1)])
def test_how_far_a_nan_reaches(dtype, T, R):
    """A NaN in v: to every query that sees it, and no further than the aligned 32 of which one
    sees a token of its block."""
    n, at = 400, 397
    cache = filled(25, 1, 1, 448, 64, [n])
    q = make(26, 1, T, R, 64, dtype=dtype)
    clean = quant_cache_attention(cache, q)[0].flatten(0, 1)
    cache.v.view(torch.uint8)[0, 0, at, 9] = 0x7f
    o = quant_cache_attention(cache, q)[0].flatten(0, 1)
    last = n - T + torch.arange(T * R, device=DEV) // R
    assert o[last >= at, 9].isnan().all()
    group = torch.arange(T * R, device=DEV) // 32
    near = torch.zeros(int(group[-1]) + 1, dtype=torch.int64, device=DEV)
    near = near.scatter_reduce(0, group, last, "amax")[group] >= at // BLOCK * BLOCK
    assert near.any() and not near.all()
    assert torch.equal(o[~near], clean[~near])
    o[:, 9] = clean[:, 9] = 0
    assert torch.equal(o, clean)


@pytest.mark.parametrize("T", [3, 50])
def test_views(T):
    B, H, G, D = 2, 4, 2, 64
    cache = filled(16, B, G, 192, D, [150, 192])
    fused = make(17, B, T, (H + 2 * G) * D)
    for q in (fused[..., :H * D].unflatten(-1, (H, D)), make(18, B, H, T, D).transpose(1, 2),
              make(19, B, T, H, D + 3)[..., 3:], make(20, 1, T, 1, D).expand(B, T, H, D),
              make(21, B * T * H * D + 1)[1:].view(B, T, H, D), make(22, 2 * B, 2 * T, H, D)[::2, ::2]):
        want = quant_cache_attention(cache, q.contiguous().clone())
        n = torch.tensor([2 ** 40, T], device=DEV)
        assert torch.equal(quant_cache_attention(cache, q), want)
        assert torch.equal(quant_cache_attention(cache, q, lengths=n), want)


def test_offsets_past_32_bits():
    """A row of 2^24 + 64 tokens in 2.2 GB of codes each: one query, and a chunk, against its last head."""
    slots, G, D = 2 ** 24 + 64, 1, 128
    codes = torch.zeros(1, G, slots, D, dtype=torch.uint8, device=DEV)
    cache = QuantCache(codes.view(E4M3), codes.clone().view(E4M3), torch.ones(1, G, slots // 64, device=DEV),
                       torch.ones(1, G, slots // 64, device=DEV),
                       torch.tensor([slots], dtype=torch.int32, device=DEV))
    assert cache.k.numel() > 2 ** 31
    tail = filled(23, 1, G, 128, D, [128])
    cache.k.view(torch.uint8)[:, :, -128:] = tail.k.view(torch.uint8)
    cache.v.view(torch.uint8)[:, :, -128:] = tail.v.view(torch.uint8)
    # the tail's keys stand out of zeros: its weight is all but exp(-100)
    for T in (1, 40):
        q = make(24, 1, T, 1, D) * 0
        q[..., 0] = 64.0
        cache.k[:, :, -128:, 0] = 448.0
        o = quant_cache_attention(cache, q, 0.01)
        for t in range(T):
            n = 128 - T + t + 1
            mean = cache.v[0, 0, -128:][:n].float().double().mean(0)
            err = (o[0, t, 0].double() - mean).abs()
            # equal scores: n equal probabilities of one rounding each, summed in fp32
            assert (err <= 2 ** -8 * mean.abs() + (2 ** -8 + 2 ** -20)
                    * cache.v[0, 0, -128:][:n].float().double().abs().mean(0)).all()
