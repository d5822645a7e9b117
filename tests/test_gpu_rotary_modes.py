"""Rotary positions in forward mode, and frequencies that ask for a gradient."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from hattention.rotary_apis import rotary_embedding, rotary_frequencies

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(seed, *shape, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=gen).to(dtype).to(DEV)


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", [(True, True), (True, False), (False, True), (True, None)])
def test_forward_mode(which, grad):
    """The map is linear: a tangent is turned as its tensor is, and one that is missing is zero."""
    freqs, _ = rotary_frequencies(24, device=DEV)
    at = torch.tensor([5, 900], device=DEV)
    turn = lambda q, k: rotary_embedding(q, k, freqs, at, "interleaved", 1.5)
    x = [make(1, 2, 6, 4, 32), None if which[1] is None else make(2, 2, 6, 2, 32)]
    d = [make(3 + i, *t.shape) if w else None for i, (t, w) in enumerate(zip(x, which))]
    plain, want = turn(*x), turn(*(t if w is None else torch.zeros_like(t) if not w else u
                                   for t, u, w in zip(x, d, which)))
    with fw.dual_level(), torch.set_grad_enabled(grad):
        y = turn(*(t if u is None else fw.make_dual(t, u) for t, u in zip(x, d)))
        for i in range(2):
            if x[i] is None:
                assert y[i] is None
                continue
            value, tangent = fw.unpack_dual(y[i])
            assert torch.equal(value, plain[i])
            assert tangent is not None and torch.equal(tangent, want[i])


def test_forward_over_backward():
    """A gradient's tangent is the tangent of what it is made from, turned back."""
    freqs, _ = rotary_frequencies(32, device=DEV)
    q, g, t = (make(i, 2, 6, 2, 32).requires_grad_(i == 1) for i in (1, 2, 3))
    with fw.dual_level():
        y, _ = rotary_embedding(q, None, freqs)
        d, = torch.autograd.grad(y, q, fw.make_dual(g, t))
        value, tangent = fw.unpack_dual(d)
    z = rotary_embedding(q, None, freqs)[0]
    assert torch.equal(value, torch.autograd.grad(z, q, g, retain_graph=True)[0])
    assert tangent is not None and torch.equal(tangent, torch.autograd.grad(z, q, t)[0])


def test_frequencies_that_require_a_gradient():
    q = make(6, 1, 4, 2, 32)
    freqs, _ = rotary_frequencies(32, device=DEV)
    freqs.requires_grad_()
    with pytest.raises(NotImplementedError, match="freqs"):
        rotary_embedding(q, None, freqs)
    with torch.no_grad():
        rotary_embedding(q, None, freqs)
    freqs = freqs.detach()
    with fw.dual_level(), pytest.raises(NotImplementedError, match="freqs"):
        rotary_embedding(q, None, fw.make_dual(freqs, freqs))
    rotary_embedding(q.requires_grad_(), None, freqs)
