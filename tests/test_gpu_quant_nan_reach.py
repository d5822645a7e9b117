"""Attention over the cache of up to 64 queries of a key head: how far a NaN in v reaches, and parts of a
row that a block of queries does not see."""
import math

import pytest
import torch

from hattention.quant_cache_apis import BLOCK, _attention_bytes, quant_cache_attention
from test_gpu_quant_attention import BF, DEV, FH, close, filled, make, oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("T,R,n,length", [
    (40, 1, 390, None), (64, 1, 130, None), (20, 2, 130, None),
    (40, 1, 1030, None),                     # the last block in a part of its own
    (64, 1, 390, 40)])                       # queries of padding behind the last
def test_how_far_a_nan_reaches(dtype, T, R, n, length):
    """To every query that sees the token, and no further than the aligned 32 of which one sees a token
    of its block."""
    at, new = n - 1, length or T
    lengths = None if length is None else torch.tensor([length], device=DEV)
    cache = filled(31, 1, 1, -(-n // BLOCK) * BLOCK, 64, [n])
    q = make(32, 1, T, R, 64, dtype=dtype)
    clean = quant_cache_attention(cache, q, lengths=lengths)[0].flatten(0, 1)
    cache.v.view(torch.uint8)[0, 0, at, 9] = 0x7f
    o = quant_cache_attention(cache, q, lengths=lengths)[0].flatten(0, 1)
    last = n - new + torch.arange(T * R, device=DEV) // R
    last[new * R:] = -1
    assert o[last >= at, 9].isnan().all()
    near = last.unflatten(0, (-1, 32)).amax(1) if T * R % 32 == 0 else \
        torch.stack([x.amax() for x in last.split(32)])
    near = near.repeat_interleave(32)[:T * R] >= at // BLOCK * BLOCK
    assert near.any() and not near.all()
    assert torch.equal(o[~near], clean[~near])
    o[:, 9] = clean[:, 9] = 0
    assert torch.equal(o, clean)


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("extra", [0, 64 * BLOCK])
def test_parts_that_a_block_does_not_see(dtype, extra):
    """Two blocks of queries whose first ends in an earlier part, rows without new tokens, and more
    queries than tokens."""
    B, T, R, D = 5, 60, 1, 64
    counts, lens = [1030, 1030, 1030, 20, 1], [60, 0, 33, 60, 32]
    cache = filled(33, B, 1, 1088 + extra, D, counts)
    q = make(34, B, T, R, D, dtype=dtype)
    for b, m in enumerate(lens):
        q[b, m:] = math.nan
    lengths = torch.tensor(lens, device=DEV)
    want, tol = oracle(cache, q, counts, lens)
    for fill in (0.0, math.nan):  # what the workspace held before is not read
        size = _attention_bytes(B, T, R, 1, D, cache.capacity)
        held = torch.full((size // 4,), fill, device=DEV)
        del held
        close(quant_cache_attention(cache, q, lengths=lengths), want, tol)
