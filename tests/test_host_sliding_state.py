"""A decoding cache of the sliding window whose attributes were set to, or made, what its kernel cannot take is
refused by the step, before any launch."""
import pytest
import torch

from hattention.sliding_apis import SlidingState, sliding_window_step

BF = torch.bfloat16


@pytest.mark.parametrize("name,change", [
    ("counts", lambda t: t - torch.ones(2, dtype=torch.int64)), ("counts", lambda t: t[:1]),
    ("counts", lambda t: torch.zeros(4, dtype=torch.int32)[::2]), ("v", lambda t: t.half()),
    ("v", lambda t: t[:, :, :8]), ("v", lambda t: t.transpose(0, 1)),
    ("k", lambda t: t.transpose(0, 1))])
@pytest.mark.parametrize("data", [False, True])
def test_sliding_state(name, change, data):
    state = SlidingState.empty(2, 2, 64, 16, 2, device="cpu")
    bad = change(getattr(state, name))
    if data:
        getattr(state, name).data = bad
    else:
        setattr(state, name, bad)
    q, k = torch.zeros(2, 4, 64, dtype=BF), torch.zeros(2, 2, 64, dtype=BF)
    with pytest.raises(ValueError):
        sliding_window_step(state, q, k, k)
