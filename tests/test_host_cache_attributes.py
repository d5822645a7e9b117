"""A cache whose attributes were set to, or made, what its kernels cannot take is refused by every call, before
any launch."""
import pytest
import torch

from hattention.quant_cache_apis import (QuantCache, quant_cache_append, quant_cache_attention,
                                         quant_cache_read, quant_cache_step)

BF = torch.bfloat16


def calls(cache):
    q, k = torch.zeros(2, 5, 4, 64, dtype=BF), torch.zeros(2, 5, 2, 64, dtype=BF)
    yield lambda: quant_cache_append(cache, k, k)
    yield lambda: quant_cache_read(cache, BF, 0, 5)
    yield lambda: quant_cache_attention(cache, q)
    yield lambda: quant_cache_step(cache, q[:, 0], k[:, 0], k[:, 0])


BAD = [
    ("counts", lambda t: t - torch.ones(2, dtype=torch.int64)), ("counts", lambda t: t[:1]),
    ("counts", lambda t: t[:, None]), ("counts", lambda t: torch.zeros(4, dtype=torch.int32)[::2]),
    ("k", lambda t: t[:, :1]), ("k", lambda t: t.float()), ("v", lambda t: t[:, :, :64]),
    ("v", lambda t: t.view(torch.uint8)), ("v", lambda t: t.transpose(0, 1)),
    ("k_scale", lambda t: t[:, :, :1]), ("k_scale", lambda t: t.double()),
    ("v_scale", lambda t: t[:1]), ("v_scale", lambda t: t.transpose(1, 2))]


@pytest.mark.parametrize("name,change", BAD)
@pytest.mark.parametrize("data", [False, True])
def test_quant_cache(name, change, data):
    cache = QuantCache.empty(2, 2, 64, 128, device="cpu")
    bad = change(getattr(cache, name))
    if data:
        getattr(cache, name).data = bad
    else:
        setattr(cache, name, bad)
    for call in calls(cache):
        with pytest.raises((ValueError, NotImplementedError)):
            call()


def test_quant_cache_that_is_set_again():
    """Attributes may be set, one after the other, as long as they fit when a call comes."""
    cache, more = (QuantCache.empty(2, 2, 64, n, device="cpu") for n in (128, 256))
    cache.counts = cache.counts - torch.ones(2, dtype=torch.int32)
    for name in ("k", "v", "k_scale", "v_scale"):
        setattr(cache, name, getattr(more, name))
        for call in calls(cache) if name != "v_scale" else ():
            with pytest.raises(ValueError):
                call()
    assert cache.capacity == 256
    for call in calls(cache):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()
