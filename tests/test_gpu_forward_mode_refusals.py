"""A hybrid stack's mixers and norm have no tangents: in forward mode they refuse, whether or not a gradient is
asked for too."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from hattention.norm_apis import layer_norm
from hattention.recurrence_apis import gated_linear_recurrence
from hattention.sliding_apis import sliding_window_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

CALLS = {
    "sliding": lambda x: sliding_window_attention(x, x.detach(), x.detach(), 4),
    "recurrence": lambda x: gated_linear_recurrence(x[0], torch.zeros_like(x[0])),
    "norm": lambda x: layer_norm(x)}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode(name, grad):
    x = torch.randn(2, 8, 2, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    if name == "recurrence":
        x = x.flatten(2)[None]
    with torch.no_grad():
        want = CALLS[name](x)
    with fw.dual_level():
        dual = fw.make_dual(x.requires_grad_(grad), torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="jvp"):
            CALLS[name](dual)
        # tensors without a tangent go through
        assert torch.equal(CALLS[name](x), want)
