"""Attention over the cache for values of v near the largest of bf16, beside others, and near the least."""
import pytest
import torch

from hattention.quant_cache_apis import BLOCK, E4M3, QuantCache, quant_cache_append, \
    quant_cache_attention, quant_cache_step
from test_gpu_quant_attention import DEV, close, make, oracle

pytestmark = pytest.mark.gpu


def near_the_top(n, T, seed, low=None):
    """A cache of n tokens in bf16 whose values reach 1.5 * 2^127, or in the first two of three blocks
    are of the sizes ``low``, and queries of its last T."""
    cache = QuantCache.empty(1, 1, 64, n, device=DEV)
    v = make(seed, 1, n, 1, 64).clamp(-3, 3) * (2.0 ** 127 / 2)
    v[0, 0, 0, 0], v[0, -1, 0, 1] = 1.5 * 2.0 ** 127, -1.5 * 2.0 ** 127
    for i, size in enumerate(low or ()):
        small = torch.arange(n, device=DEV) // BLOCK % 3 == i
        v[0, small] = make(seed + 1 + i, int(small.sum()), 1, 64) * size
    quant_cache_append(cache, make(seed + 3, 1, n, 1, 64), v)
    assert cache.v_scale.amax() == 2.0 ** 119
    return cache, make(seed + 4, 1, T, 2, 64, scale=0.5)


@pytest.mark.parametrize("n,T", [(2, 1), (2, 2), (5000, 1), (300, 30), (300, 200), (6000, 100)])
def test_values_near_the_largest(n, T):
    """Weighted means of values that are finite are finite, as far as bf16 goes: the sums over the weights,
    which come to more than 1 before they are divided, stay in range."""
    cache, q = near_the_top(n, T, 43)
    close(quant_cache_attention(cache, q), *oracle(cache, q, [n], [T]))


@pytest.mark.parametrize("H", [4, 40])
def test_values_near_the_largest_in_a_step(H):
    cache, _ = near_the_top(130, 1, 47)
    for i in range(3):
        q, k = make(50 + i, 1, H, 64, scale=0.5), make(60 + i, 1, 1, 64)
        v = k * 2.0 ** 125
        o, _ = quant_cache_step(cache, q, k, v)
        close(o[:, None], *oracle(cache, q[:, None], [131 + i], [1]))


@pytest.mark.parametrize("n,T", [(700, 1), (700, 40), (700, 300), (6000, 100)])
@pytest.mark.parametrize("low", [(1.0, 1.0), (2.0 ** -40, 2.0 ** -40), (2.0 ** 60, 2.0 ** 60),
                                 (2.0 ** -70, 1.0)])  # the first are as good as zeros, with a weight
def test_values_of_very_different_sizes(n, T, low):
    """Blocks near the largest value beside ordinary ones: queries whose weights all lie on the small ones
    keep them, whatever came before."""
    cache, q = near_the_top(n, T, 53, low)
    close(quant_cache_attention(cache, q), *oracle(cache, q, [n], [T]))
    # a first coordinate of keys and queries that hides the large blocks from every query
    large = torch.arange(n, device=DEV) // BLOCK % 3 == 2
    cache.k[0, 0, :n, 0] = torch.where(large, -448.0, 448.0).to(E4M3)
    q[..., 0] = 256.0
    o = quant_cache_attention(cache, q, 1.0)
    want, tol = oracle(cache, q, [n], [T], 1.0)
    assert want.abs().amax() < max(low) * 8
    close(o, want, tol)


@pytest.mark.parametrize("T", [1, 40, 200])
def test_small_values(T):
    """Values at the least scale are kept."""
    n = 700
    cache = QuantCache.empty(1, 1, 64, n, device=DEV)
    v = make(57, 1, n, 1, 64) * 2.0 ** -93
    quant_cache_append(cache, make(58, 1, n, 1, 64), v)
    assert cache.v_scale[..., :n // BLOCK].amax() <= 2.0 ** -98
    q = make(59, 1, T, 2, 64)
    close(quant_cache_attention(cache, q), *oracle(cache, q, [n], [T]))
