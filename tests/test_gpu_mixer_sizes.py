"""The largest launches that the mixers' size checks let through: just under 2^32 threads."""
import pytest
import torch

from hattention.recurrence_apis import gated_linear_recurrence, gated_linear_recurrence_step
from hattention.sliding_apis import SlidingState, sliding_window_attention, sliding_window_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FS = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


def test_recurrence():
    B = 2 ** 23 - 1
    x = torch.randn(B, 1, 1, generator=torch.Generator(DEV).manual_seed(1), device=DEV)
    x.requires_grad_()
    o = gated_linear_recurrence(x, torch.zeros_like(x))
    assert torch.equal(o, x)
    assert torch.equal(torch.autograd.grad(o, x, x.detach())[0], x)
    with pytest.raises(NotImplementedError):
        gated_linear_recurrence(torch.zeros(B + 1, 1, 1, device=DEV),
                                torch.zeros(B + 1, 1, 1, device=DEV))


def test_recurrence_step():
    B, D = 2 ** 16, 2 ** 16 - 1
    h = torch.ones(B, D, device=DEV)
    x, g = torch.full((B, D), 2.0, device=DEV, dtype=BF), torch.zeros(B, D, device=DEV, dtype=BF)
    o, h = gated_linear_recurrence_step(h, x, g)
    for t in (o, h):
        assert float(t.amin()) == float(t.amax()) == 3.0


def test_attention():
    B, H = 2 ** 13 - 1, 2 ** 11  # 2^24 - 2^11 workgroups
    q = torch.zeros(B, 1, H, 8, device=DEV, dtype=BF)
    v = torch.randn(B, 1, 1, 8, generator=torch.Generator(DEV).manual_seed(1), device=DEV).to(BF)
    o = sliding_window_attention(q, v, v, 4)
    assert torch.equal(o, v.expand_as(o))


def test_attention_step():
    B, H = 2 ** 21 - 1, 16  # 2^25 - 16 rows of 128 threads
    state = SlidingState.empty(B, 1, 8, 1, device=DEV)
    q = torch.zeros(B, H, 8, device=DEV, dtype=BF)
    v = torch.randn(B, 1, 8, generator=torch.Generator(DEV).manual_seed(1), device=DEV).to(BF)
    o, state = sliding_window_step(state, q, v, v)
    assert torch.equal(o, v.expand_as(o)) and torch.equal(state.v[:, :, 0], v)
    assert int(state.counts.amin()) == int(state.counts.amax()) == 1
