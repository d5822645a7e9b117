"""Outputs and gradients past a row's length are zero, also where a token of the row is not finite."""
import pytest
import torch

from hattention.sliding_apis import sliding_window_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NAN, INF = float("nan"), float("inf")


def make(seed, *shape, dtype=torch.bfloat16):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=gen).to(dtype).to(DEV)


@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (128, torch.float16), (80, torch.bfloat16)])
@pytest.mark.parametrize("n,W,S", [(140, 50, 4), (140, 200, 0), (2, 1, 4), (2, 50, 33), (1, 1, 0),
                                   (257, 100, 64)])
@pytest.mark.parametrize("where", ["q", "k", "v", "do"])
def test_zero_past_the_length(D, dtype, n, W, S, where):
    B, T, H, G = 2, 400, 4, 2
    x = {"q": make(1, B, T, H, D, dtype=dtype), "k": make(2, B, T, G, D, dtype=dtype),
         "v": make(3, B, T, G, D, dtype=dtype), "do": make(4, B, T, H, D, dtype=dtype)}
    x[where][1, n - 1] = NAN
    x[where][1, 0, 0, :3] = INF
    do, leaves = x.pop("do"), [t.requires_grad_() for t in x.values()]
    lengths = torch.tensor([T, n], dtype=torch.int32, device=DEV)
    o = sliding_window_attention(*leaves, W, S, lengths=lengths)
    grads = torch.autograd.grad(o, leaves, do)
    for name, t in zip(["o", "dq", "dk", "dv"], [o.detach(), *grads]):
        assert (t[1, n:] == 0).all(), (name, t[1, n:].isnan().sum().item())
        assert t[0].isfinite().all(), name
    with torch.no_grad():
        assert (sliding_window_attention(*leaves, W, S, lengths=lengths)[1, n:] == 0).all()
