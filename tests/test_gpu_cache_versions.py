"""Caches are advanced in place, which autograd is told: positions that are taken from their counts and advanced
between a forward and its backward."""
import pytest
import torch

from hattention.quant_cache_apis import QuantCache, quant_cache_append, quant_cache_step
from hattention.recurrence_apis import gated_linear_recurrence_step
from hattention.rotary_apis import rotary_embedding, rotary_frequencies
from hattention.sliding_apis import SlidingState, sliding_window_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(seed, *shape, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=gen).to(dtype).to(DEV)


@pytest.mark.parametrize("how", ["append", "step"])
def test_counts_advanced_before_the_backward(how):
    """Positions taken from a cache's counts, which tokens then advance: the backward refuses, as after any
    change in place, and a copy of them works."""
    freqs, _ = rotary_frequencies(64, device=DEV)
    cache = QuantCache.empty(2, 1, 64, 64, device=DEV)
    q, k = make(4, 2, 3, 2, 64).requires_grad_(), make(5, 2, 3, 1, 64, dtype=torch.bfloat16)

    def advance():
        if how == "append":
            quant_cache_append(cache, k, k)
        else:
            quant_cache_step(cache, k[:, 0].expand(2, 2, 64), k[:, 0], k[:, 0])

    advance()
    want = torch.autograd.grad(rotary_embedding(q, None, freqs, cache.counts)[0].sum(), q)[0]
    y, _ = rotary_embedding(q, None, freqs, cache.counts)
    z, _ = rotary_embedding(q, None, freqs, cache.counts.clone())
    before = [t._version for t in cache._tensors()]
    advance()
    assert all(t._version > n for t, n in zip(cache._tensors(), before))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    assert torch.equal(torch.autograd.grad(z.sum(), q)[0], want)


def test_a_sliding_cache_advanced_before_the_backward():
    freqs, _ = rotary_frequencies(64, device=DEV)
    state = SlidingState.empty(2, 1, 64, 16, 2, device=DEV)
    q, k = make(6, 2, 2, 64).requires_grad_(), make(7, 2, 1, 64, dtype=torch.bfloat16)
    y, _ = rotary_embedding(q, None, freqs, state.counts)
    sliding_window_step(state, k.expand(2, 2, 64).contiguous(), k, k)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_a_recurrence_advanced_before_the_backward():
    state = torch.zeros(2, 64, device=DEV)
    x = make(9, 2, 64).requires_grad_()
    y = x * state
    gated_linear_recurrence_step(state, x.detach(), x.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_caches_of_inference_mode():
    """They have no version, and are advanced in and out of that mode."""
    with torch.inference_mode():
        cache = QuantCache.empty(1, 1, 64, 64, device=DEV)
        state = SlidingState.empty(1, 1, 64, 16, device=DEV)
    x = make(8, 1, 1, 64, dtype=torch.bfloat16)
    for mode in (True, False):
        with torch.inference_mode(mode):
            quant_cache_append(cache, x[:, None], x[:, None])
            quant_cache_step(cache, x, x, x)
            sliding_window_step(state, x, x, x)
    assert cache.counts.tolist() == [4] and state.counts.tolist() == [2]
