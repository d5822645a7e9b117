"""Rotary positions against the formula in 64 bits, and gradients against it and differences.

Tolerance: a sine and a cosine carry at most 4 u (two units of the function, the argument's
rounding of at most pi u, u = 2^-24, and the product with the scale), the two products and their
sum 2 u more: 6 u scale (|a| + |b|), twice that where u of the result is rounded up; then the
half step of the result's type.  The position times its frequency has 64 bits: 2^-51 of the angle.
"""
import pytest
import torch

from hattention.rotary_apis import rotary_embedding, rotary_frequencies

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
BF, FH, FS = torch.bfloat16, torch.float16, torch.float32


def make(seed, *shape, dtype=BF):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=gen).to(dtype).to(DEV)


def halves(x, n, layout):
    if layout == "half":
        return x[..., :n], x[..., n:2 * n]
    return x[..., 0:2 * n:2], x[..., 1:2 * n:2]


def oracle(x, freqs, at, layout, scale=1.0, back=False):
    """(result, bound) for x [B, T, heads, D] at positions at [B, T]."""
    n, y = freqs.shape[0], x.double().clone()
    tol = torch.zeros_like(y)
    angle = (at.double()[..., None] * freqs.double())[:, :, None]
    cos, sin = torch.cos(angle) * scale, torch.sin(angle) * (-scale if back else scale)
    a, b = halves(x.double(), n, layout)
    ya, yb = halves(y, n, layout)
    ya.copy_(a * cos - b * sin)
    yb.copy_(a * sin + b * cos)
    for t in halves(tol, n, layout):
        t.copy_((12 * U + 2.0 ** -51 * angle.abs()) * abs(scale) * (a.abs() + b.abs()))
    return y, tol


def close(got, want, tol):
    f = torch.finfo(got.dtype)
    tol = tol + f.eps / 2 * (want.abs() + tol) + f.smallest_normal * f.eps
    over = (got.double() - want).abs() - tol
    assert not (over > 0).any(), float(over.max())


def positions(kind, B, T, far=0, dtype=torch.int64):
    t = torch.arange(T, device=DEV)
    if kind == "none":
        return None, t.expand(B, T)
    if kind == "row":
        first = torch.tensor([far + 37 * b for b in range(B)], device=DEV)
        return first.to(dtype), first[:, None] + t
    at = far + (t * 7919 + torch.arange(B, device=DEV)[:, None] * 31) % (T + 50)
    return at.to(dtype), at


@pytest.mark.parametrize("dtype", [BF, FH, FS])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("B,T,H,G,D,n", [
    (1, 1, 1, 1, 2, 1), (2, 37, 4, 2, 64, 32), (3, 5, 6, 1, 128, 16), (1, 300, 2, 2, 80, 40),
    (2, 9, 3, 3, 96, 20), (1, 7, 1, 1, 33, 7), (2, 3, 5, 1, 256, 128), (1, 2, 2, 2, 512, 256),
    (1, 3, 2, 1, 512, 1), (2, 65, 40, 8, 32, 16), (1, 4000, 3, 1, 16, 8), (1, 2, 300, 7, 8, 4),
    (1, 3, 2, 2, 24, 8), (1, 3, 2, 2, 20, 8)])
def test_forward_and_backward(dtype, layout, B, T, H, G, D, n):
    q, k = make(1, B, T, H, D, dtype=dtype), make(2, B, T, G, D, dtype=dtype)
    freqs = torch.rand(n, dtype=torch.float64, generator=torch.Generator().manual_seed(n)).to(DEV)
    for kind, scale in (("none", 1.0), ("row", 1.25), ("token", 1.0)):
        pos, at = positions(kind, B, T)
        x = [t.clone().requires_grad_() for t in (q, k)]
        y = rotary_embedding(*x, freqs, pos, layout, scale)
        g = [make(5 + i, *t.shape, dtype=dtype) for i, t in enumerate(y)]
        d = torch.autograd.grad(y, x, g)
        for i in range(2):
            assert y[i].dtype == dtype and y[i].is_contiguous()
            close(y[i].detach(), *oracle(x[i].detach(), freqs, at, layout, scale))
            close(d[i], *oracle(g[i], freqs, at, layout, scale, back=True))
        with torch.no_grad():
            z = rotary_embedding(q, k, freqs, pos, layout, scale)
            assert all(torch.equal(a, b) for a, b in zip(y, z))
            assert torch.equal(rotary_embedding(q, None, freqs, pos, layout, scale)[0], y[0])


@pytest.mark.parametrize("far", [2 ** 20, 2 ** 31 - 400, 2 ** 40, -2 ** 31])
def test_far_positions(far):
    q = make(3, 2, 300, 2, 64, dtype=FS)
    freqs, _ = rotary_frequencies(64, device=DEV)
    for kind in ("row", "token"):
        for dtype in (torch.int32, torch.int64):
            if dtype == torch.int32 and abs(far) > 2 ** 31:
                continue
            pos, at = positions(kind, 2, 300, far, dtype)
            y, _ = rotary_embedding(q, None, freqs, pos)
            close(y, *oracle(q, freqs, at, "half"))


def test_frequencies_in_32_bits_and_positions_with_strides():
    q, k = make(4, 3, 6, 2, 32, dtype=FS), make(5, 3, 6, 1, 32, dtype=FS)
    freqs = rotary_frequencies(32, device=DEV)[0].float()
    at = torch.arange(36, device=DEV, dtype=torch.int32).view(6, 6)
    for pos in (at.t()[:3], at[:1].expand(3, 6), at[:3, :1].expand(3, 6), at[:3, ::1]):
        y = rotary_embedding(q, k, freqs, pos)
        for i, x in enumerate((q, k)):
            close(y[i], *oracle(x, freqs, pos, "half"))
    spread = at[0, ::2]  # [3], every other one
    y = rotary_embedding(q, k, freqs, spread)[0]
    close(y, *oracle(q, freqs, spread[:, None] + torch.arange(6, device=DEV), "half"))
    twice = torch.stack([freqs, freqs], 1)[:, 0]  # not contiguous
    assert torch.equal(rotary_embedding(q, k, twice, spread)[0], y)


def views(dtype, B=2, T=9, H=4, G=2, D=64):
    """q and k as a caller may hold them."""
    fused = make(6, B, T, (H + 2 * G) * D, dtype=dtype)
    yield (fused[..., :H * D].unflatten(-1, (H, D)), fused[..., H * D:(H + G) * D].unflatten(-1, (G, D)))
    heads = make(7, B, H + G, T, D, dtype=dtype).transpose(1, 2)
    yield heads[:, :, :H], heads[:, :, H:]
    odd = make(8, B * T * (H + G) * D + 1, dtype=dtype)[1:].view(B, T, H + G, D)  # off 16 bytes
    yield odd[:, :, :H], odd[:, :, H:]
    wide = make(9, B, T, H + G, D + 1, dtype=dtype)[..., 1:]
    yield wide[:, :, :H], wide[:, :, H:]
    last = make(10, B, T, D, H + G, dtype=dtype).transpose(2, 3)
    yield last[:, :, :H], last[:, :, H:]
    one = make(11, B, 1, 1, D, dtype=dtype)
    yield one.expand(B, T, H, D), one.expand(B, T, G, D)


@pytest.mark.parametrize("dtype", [BF, FS])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_views(dtype, layout):
    freqs, _ = rotary_frequencies(32, device=DEV)
    for q, k in views(dtype):
        x = [q.detach().requires_grad_(), k.detach().requires_grad_()]
        y = rotary_embedding(*x, freqs, None, layout)
        z = rotary_embedding(q.contiguous(), k.contiguous(), freqs, None, layout)
        assert all(torch.equal(a, b) for a, b in zip(y, z))
        # gradients that come as views too
        g = [t.detach() for t in (q, k)]
        d = torch.autograd.grad(y, x, g)
        at = torch.arange(q.shape[1], device=DEV).expand(q.shape[:2])
        for i in range(2):
            close(d[i], *oracle(g[i], freqs, at, layout, back=True))


def test_which_gradients():
    q, k = make(1, 2, 5, 2, 32, dtype=FS), make(2, 2, 5, 1, 32, dtype=FS)
    freqs, _ = rotary_frequencies(32, device=DEV)
    full = [t.clone().requires_grad_() for t in (q, k)]
    y = rotary_embedding(*full, freqs)
    dq, dk = torch.autograd.grad(y[0].sum() + y[1].sum(), full)
    for i, want in ((0, dq), (1, dk)):
        x = [t.clone() for t in (q, k)]
        x[i].requires_grad_()
        y = rotary_embedding(*x, freqs)
        assert torch.equal(torch.autograd.grad(y[i].sum(), x[i])[0], want)
        # only one of the outputs is used
        y = rotary_embedding(*[t.detach().requires_grad_() for t in (q, k)], freqs)
        leaf = full[i].detach().requires_grad_()
        pair = [leaf if j == i else t for j, t in enumerate((q, k))]
        y = rotary_embedding(*pair, freqs)
        assert torch.equal(torch.autograd.grad(y[i].sum(), leaf)[0], want)
    x = [t.clone().requires_grad_() for t in (q, k)]
    y = rotary_embedding(*x, freqs)
    got = torch.autograd.grad(y[0].sum(), x, allow_unused=True)
    assert torch.equal(got[0], dq) and got[1] is None
    x = q.clone().requires_grad_()
    y, none = rotary_embedding(x, None, freqs)
    assert none is None and torch.equal(torch.autograd.grad(y.sum(), x)[0], dq)


def test_gradient_of_the_gradient():
    """The gradient turns back, its own gradient forth."""
    q, k = make(1, 2, 5, 2, 32, dtype=FS).requires_grad_(), make(2, 2, 5, 1, 32, dtype=FS).requires_grad_()
    g = [t.detach().clone().requires_grad_() for t in (make(3, 2, 5, 2, 32, dtype=FS),
                                                        make(4, 2, 5, 1, 32, dtype=FS))]
    freqs, _ = rotary_frequencies(32, device=DEV)
    y = rotary_embedding(q, k, freqs, None, "half", 1.5)
    d = torch.autograd.grad(y, [q, k], g, create_graph=True)
    h = [make(5, 2, 5, 2, 32, dtype=FS), make(6, 2, 5, 1, 32, dtype=FS)]
    dd = torch.autograd.grad(d, g, h)
    at = torch.arange(5, device=DEV).expand(2, 5)
    for i in range(2):
        close(dd[i], *oracle(h[i], freqs, at, "half", 1.5))


def test_gradient_against_differences():
    """The map is linear, so its difference along any direction is the gradient along it."""
    q = make(1, 1, 6, 2, 32, dtype=FS).requires_grad_()
    freqs, _ = rotary_frequencies(24, device=DEV)
    at = torch.tensor([1000], device=DEV)
    g = make(2, 1, 6, 2, 32, dtype=FS)
    step = make(3, 1, 6, 2, 32, dtype=FS)
    y, _ = rotary_embedding(q, None, freqs, at, "interleaved", 1.5)
    d = torch.autograd.grad(y, q, g)[0].double()
    with torch.no_grad():
        z, _ = rotary_embedding(q + step, None, freqs, at, "interleaved", 1.5)
        moved = (z.double() - y.double()) * g.double()
        # each result is off by 13 u 1.5 (|a| + |b|), and q + step by u
        size = float(((q.abs() + step.abs()).double().sum() * 1.5 * g.double().abs().amax()))
        assert abs(float((d * step.double()).sum() - moved.sum())) < 4 * 14 * U * 2 * size


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_one_token(layout):
    q, k = make(1, 5, 6, 64), make(2, 5, 2, 64)
    freqs, _ = rotary_frequencies(64, device=DEV)
    at = torch.tensor([0, 1, 700, 123456, 2 ** 20], device=DEV, dtype=torch.int32)
    y = rotary_embedding(q, k, freqs, at, layout)
    for i, x in enumerate((q, k)):
        assert y[i].shape == x.shape
        close(y[i].unsqueeze(1), *oracle(x.unsqueeze(1), freqs, at[:, None], layout))
    x = [t.clone().requires_grad_() for t in (q, k)]
    z = rotary_embedding(*x, freqs, at, layout)
    d = torch.autograd.grad(z, x, [q, k])
    close(d[0].unsqueeze(1), *oracle(q.unsqueeze(1), freqs, at[:, None], layout, back=True))


def test_what_is_not_finite_stays_in_its_pair():
    q = make(1, 1, 3, 2, 32, dtype=FS)
    q[0, 1, 1, 4] = float("nan")
    q[0, 2, 0, 30] = float("inf")  # beyond the rotated part
    freqs, _ = rotary_frequencies(24, device=DEV)
    y, _ = rotary_embedding(q, None, freqs)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[0, 1, 1, 4] = bad[0, 1, 1, 16] = True
    assert torch.equal(y.isnan(), bad)
    assert y[0, 2, 0, 30] == float("inf") and (y.isfinite() == ~(bad | y.isinf())).all()


def test_offsets_past_32_bits():
    """2.2 G elements: the last tokens, and the first."""
    T, H, D = 33600, 512, 128
    q = torch.zeros(1, T, H, D, dtype=BF, device=DEV)
    ends = [0, 1, T - 2, T - 1]
    q[:, ends] = make(1, 1, 4, H, D)
    assert q.numel() > 2 ** 31
    freqs, _ = rotary_frequencies(D, device=DEV)
    y, _ = rotary_embedding(q, None, freqs)
    close(y[:, ends], *oracle(q[:, ends], freqs, torch.tensor([ends], device=DEV), "half"))
    assert not y[:, 2:-2].any()
