"""Attention over the cache where the product of the scales of the keys and of the scores is 0 in 32 bits."""
import pytest
import torch

from hattention.quant_cache_apis import QuantCache, quant_cache_append, quant_cache_attention
from test_gpu_quant_attention import BF, DEV, FH, close, make, oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("T", [1, 40, 200])
@pytest.mark.parametrize("scale", [1e-30, 1e-12])
def test_scores_of_no_size(dtype, T, scale):
    """Keys of zero, whose blocks have the least scale there is, and a scale of the scores for which the
    product of both is 0 in 32 bits, or all but: every token that a query sees weighs the same."""
    n = 230
    cache = QuantCache.empty(1, 1, 64, 256, device=DEV)
    v = make(41, 1, n, 1, 64, dtype=dtype)
    quant_cache_append(cache, torch.zeros_like(v), v)
    assert (cache.k_scale[..., 0] == 2.0 ** -100).all()
    q = make(42, 1, T, 2, 64, dtype=dtype)
    close(quant_cache_attention(cache, q, scale), *oracle(cache, q, [n], [T], scale))
    # and NaN in a key stays NaN where it is seen
    cache.k.view(torch.uint8)[0, 0, n - 1, 3] = 0x7f
    o = quant_cache_attention(cache, q, scale)
    assert o[0, -1].isnan().all() and o[0, :-1].isfinite().all()
