"""Attention over a cache whose codes lie past 2^31 bytes, in blocks of many queries."""
import pytest
import torch

from hattention.quant_cache_apis import BLOCK, E4M3, QuantCache, quant_cache_attention
from test_gpu_quant_attention import BF, DEV, filled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [70, 127])
def test_offsets_past_32_bits(T):
    """A row of 2^24 + 64 tokens in 2.2 GB of codes each, and a block of many queries at its end, against
    the last tokens, which stand out of zeros: the others weigh exp(-100) and less."""
    slots, D = 2 ** 24 + 64, 128
    codes = torch.zeros(1, 1, slots, D, dtype=torch.uint8, device=DEV)
    one = torch.ones(1, 1, slots // BLOCK, device=DEV)
    cache = QuantCache(codes.view(E4M3), codes.clone().view(E4M3), one, one.clone(),
                       torch.tensor([slots], dtype=torch.int32, device=DEV))
    assert cache.k.numel() > 2 ** 31
    cache.v[:, :, -128:] = filled(23, 1, 1, 128, D, [128]).v
    cache.k[:, :, -128:, 0] = 448.0
    q = torch.zeros(1, T, 1, D, dtype=BF, device=DEV)
    q[..., 0] = 64.0
    o = quant_cache_attention(cache, q, 0.01)
    v = cache.v[0, 0, -128:].float().double()
    for t in range(T):
        seen = v[:128 - T + t + 1]
        err = (o[0, t, 0].double() - seen.mean(0)).abs()
        # equal scores: equal probabilities of one rounding each, summed in fp32, and the result's own
        assert (err <= 2 ** -8 * seen.mean(0).abs() + (2 ** -8 + 2 ** -20) * seen.abs().mean(0)).all()
