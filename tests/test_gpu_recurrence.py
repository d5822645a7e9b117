"""gated_linear_recurrence against the token loop in 64 bits.

Tolerances: every token multiplies and adds in fp32 (u = 2^-24) and takes exp(g), whose
argument is scaled by log2(e) and so errs by |g| u.  With habs_t = a_t habs_{t-1} + |x_t|
the error obeys e_t <= a_t e_{t-1} + c (1 + |g_t|) u habs_t; the maps of a wave, a segment and
the walk over the segments add as many roundings again, each of the same magnitudes: c = 16.
The result's own half step comes on top.
"""
import pytest
import torch

from hattention.recurrence_apis import gated_linear_recurrence, gated_linear_recurrence_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
BF, FH, FS = torch.bfloat16, torch.float16, torch.float32


def make(seed, *shape, dtype=FS, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * scale).to(dtype).to(DEV)


def gates(seed, B, T, D, dtype):
    gen = torch.Generator().manual_seed(seed)
    rate = torch.exp(-torch.rand(D, generator=gen) * 7)
    return (-rate * torch.exp(torch.randn(B, T, D, generator=gen) * 0.5)).to(dtype).to(DEV)


def scan(a, b, start, live):
    h, out = start, []
    for t in range(a.shape[1]):
        h = torch.where(live[:, t], a[:, t] * h + b[:, t], h)
        out.append(h)
    return torch.stack(out, 1), h


def oracle(x, g, h0, lengths, do=None, dht=None):
    """(results, bounds) in 64 bits; on the CPU, token by token."""
    x, g = x.double().cpu(), g.double().cpu()
    B, T, D = x.shape
    n = lengths.cpu() if lengths is not None else torch.full((B,), T)
    live = torch.arange(T)[None, :, None] < n.clamp(0, T)[:, None, None]
    a = torch.exp(g)
    zero = torch.zeros(B, D, dtype=torch.float64)
    h0 = h0.double().cpu() if h0 is not None else zero
    c = 16 * U * (1 + torch.where(a > 0, g.abs(), 0.0))
    h, ht = scan(a, x, h0, live)
    habs, _ = scan(a, x.abs(), h0.abs(), live)
    e, et = scan(a, c * habs, zero, live)
    mask = lambda z: torch.where(live, z, 0.0)
    out, tol = {"o": mask(h), "ht": ht}, {"o": mask(e), "ht": et}
    if do is not None:
        do = mask(do.double().cpu())
        dht = dht.double().cpu() if dht is not None else zero
        d, dabs, de = dht, dht.abs(), zero
        dh, eh, ab = [None] * T, [None] * T, [None] * T
        for t in range(T - 1, -1, -1):
            lv = live[:, t]
            dh[t], ab[t] = do[:, t] + d, do[:, t].abs() + dabs
            eh[t] = de + c[:, t] * ab[t]
            d = torch.where(lv, a[:, t] * dh[t], d)
            dabs = torch.where(lv, a[:, t] * ab[t], dabs)
            de = torch.where(lv, a[:, t] * eh[t] + c[:, t] * a[:, t] * ab[t], de)
        dh, eh = mask(torch.stack(dh, 1)), mask(torch.stack(eh, 1))
        prev = lambda z, s: torch.cat([s[:, None], z[:, :-1]], 1)
        hp, ep = prev(h, h0), prev(e, zero)
        out.update(dx=dh, dg=mask(dh * a * hp), dh0=d)
        tol.update(dx=eh, dg=mask(a * (eh * hp.abs() + dh.abs() * ep) + c * (dh * a * hp).abs()),
                   dh0=de)
    return out, tol


def close(name, got, want, tol):
    got, half = got.detach().cpu(), torch.finfo(got.dtype).eps / 2
    d = (got.double() - want).abs()
    lim = tol + half * (want.abs() + tol) + torch.finfo(got.dtype).smallest_normal
    bad = ~(d <= lim)
    assert not bad.any(), (name, float(d.max()), float((d / lim).max()))


CASES = [  # B, T, D, x, g, state, lengths
    (1, 1, 1, FS, FS, False, None), (2, 1, 70, BF, BF, True, None), (1, 31, 64, FH, FS, True, None),
    (2, 32, 65, BF, FS, False, [32, 0]), (1, 33, 3, FS, FS, True, None),
    (2, 255, 129, BF, BF, True, [255, 1]), (1, 256, 64, FH, FH, True, None),
    (3, 257, 40, FS, FS, True, [257, 256, 255]), (2, 700, 100, BF, FS, True, [33, 700]),
    (1, 2600, 66, FS, FS, False, None), (2, 3000, 64, BF, BF, True, [2999, -5]),
    (1, 1000, 64, FH, FS, False, [5000]), (1, 6000, 8, FS, FS, True, None),
]


@pytest.mark.parametrize("B,T,D,xt,gt,state,lens", CASES)
def test_forward_and_gradients(B, T, D, xt, gt, state, lens):
    x = make(1, B, T, D, dtype=xt).requires_grad_()
    g = gates(2, B, T, D, gt).requires_grad_()
    h0 = make(3, B, D, scale=2.0).requires_grad_() if state else None
    n = torch.tensor(lens, dtype=torch.int32, device=DEV) if lens else None
    do, dht = make(4, B, T, D, dtype=xt), make(5, B, D)
    o, ht = gated_linear_recurrence(x, g, h0, True, n)
    leaves = [x, g] + ([h0] if state else [])
    grads = torch.autograd.grad([o, ht], leaves, [do, dht])
    want, tol = oracle(x.detach(), g.detach(), h0.detach() if state else None, n, do, dht)
    for name, got in zip(["o", "ht", "dx", "dg", "dh0"], [o, ht, *grads]):
        close(name, got, want[name], tol[name])
    with torch.no_grad():
        o2, ht2 = gated_linear_recurrence(x, g, h0, True, n)
    assert torch.equal(o2, o) and torch.equal(ht2, ht)


def test_same_bits_every_time():
    """Where a walk over the segments begins depends on time; the result does not."""
    x, g = make(1, 2, 20000, 192, dtype=BF), gates(2, 2, 20000, 192, BF)
    first = gated_linear_recurrence(x, g, None, True)
    for _ in range(5):
        again = gated_linear_recurrence(x, g, None, True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    xg, gg = x.clone().requires_grad_(), g.clone().requires_grad_()
    do = make(3, 2, 20000, 192, dtype=BF)
    base = None
    for _ in range(4):
        got = torch.autograd.grad(gated_linear_recurrence(xg, gg), [xg, gg], do)
        base = base or got
        assert all(torch.equal(p, q) for p, q in zip(base, got))


def test_long_memory():
    """Decays near one: the state of the first tokens reaches the last of many segments."""
    B, T, D = 1, 9000, 64
    x = make(1, B, T, D)
    g = torch.full((B, T, D), -1e-4, device=DEV)
    o, ht = gated_linear_recurrence(x, g, None, True)
    want, tol = oracle(x, g, None, None)
    close("o", o, want["o"], tol["o"])
    close("ht", ht, want["ht"], tol["ht"])


def test_resets():
    """g = -inf forgets what was before, also across segments and in the gradient."""
    B, T, D = 1, 1200, 64
    x = make(1, B, T, D).requires_grad_()
    g0 = gates(2, B, T, D, FS)
    g0[:, [0, 100, 256, 777]] = -float("inf")
    g0[:, 300, :10] = -200.0  # underflows to zero
    g = g0.requires_grad_()
    do = make(3, B, T, D)
    o = gated_linear_recurrence(x, g)
    dx, dg = torch.autograd.grad(o, [x, g], do)
    want, tol = oracle(x.detach(), g.detach(), None, None, do)
    close("o", o, want["o"], tol["o"])
    close("dx", dx, want["dx"], tol["dx"])
    close("dg", dg, want["dg"], tol["dg"])
    assert torch.equal(o[:, 256].detach(), x[:, 256].detach())


def test_padding_is_not_read():
    B, T, D = 2, 600, 65
    x, g = make(1, B, T, D, dtype=BF), gates(2, B, T, D, BF)
    n = torch.tensor([600, 300], device=DEV)
    o, ht = gated_linear_recurrence(x, g, None, True, n)
    x2, g2 = x.clone(), g.clone()
    x2[1, 300:], g2[1, 300:] = float("nan"), float("inf")
    x2.requires_grad_(), g2.requires_grad_()
    o2, ht2 = gated_linear_recurrence(x2, g2, None, True, n)
    assert torch.equal(o, o2) and torch.equal(ht, ht2)
    do = make(3, B, T, D, dtype=BF)
    do[1, 300:] = float("nan")
    dx, dg = torch.autograd.grad(o2, [x2, g2], do)
    assert dx.isfinite().all() and dg.isfinite().all()
    assert not dx[1, 300:].any() and not dg[1, 300:].any()


def test_nan_stays_in_its_channel():
    B, T, D = 1, 900, 70
    x, g = make(1, B, T, D), gates(2, B, T, D, FS)
    o = gated_linear_recurrence(x, g)
    x2 = x.clone()
    x2[0, 400, 3] = float("nan")
    o2 = gated_linear_recurrence(x2, g)
    keep = [d for d in range(D) if d != 3]
    assert torch.equal(o[..., keep], o2[..., keep]) and torch.equal(o[:, :400], o2[:, :400])
    assert o2[0, 400:, 3].isnan().all()


def test_continuing_from_a_state():
    """Two calls joined by the state give one call's result, gradients too."""
    B, T, D, cut = 2, 800, 96, 333
    x, g = make(1, B, T, D), gates(2, B, T, D, FS)
    do = make(3, B, T, D)
    leaves = [t.clone().requires_grad_() for t in (x, g)]
    a, h = gated_linear_recurrence(leaves[0][:, :cut], leaves[1][:, :cut], None, True)
    b = gated_linear_recurrence(leaves[0][:, cut:], leaves[1][:, cut:], h)
    got = torch.autograd.grad([a, b], leaves, [do[:, :cut], do[:, cut:]])
    want, tol = oracle(x, g, None, None, do)
    close("o", torch.cat([a, b], 1), want["o"], tol["o"])
    close("dx", got[0], want["dx"], tol["dx"])
    close("dg", got[1], want["dg"], tol["dg"])


def test_step():
    B, T, D = 3, 20, 130
    for xt, gt in ((BF, FS), (FH, FH), (FS, FS)):
        x, g = make(1, B, T, D, dtype=xt), gates(2, B, T, D, gt)
        h = make(3, B, D)
        want, tol = oracle(x, g, h, None)
        state = h.clone()
        for t in range(T):
            o, s = gated_linear_recurrence_step(state, x[:, t], g[:, t])
            assert s is state
            close("o", o, want["o"][:, t], tol["o"][:, t])
        close("ht", state, want["ht"], tol["ht"])


def test_only_the_final_state():
    B, T, D = 1, 300, 64
    x = make(1, B, T, D).requires_grad_()
    g = gates(2, B, T, D, FS)
    _, ht = gated_linear_recurrence(x, g, None, True)
    dht = make(3, B, D)
    (dx,) = torch.autograd.grad(ht, [x], dht)
    want, tol = oracle(x.detach(), g, None, None, torch.zeros(B, T, D, device=DEV), dht)
    close("dx", dx, want["dx"], tol["dx"])


def test_difference_quotient():
    B, T, D = 1, 40, 2
    x, g = make(1, B, T, D).requires_grad_(), gates(2, B, T, D, FS).requires_grad_()
    do = make(3, B, T, D)
    dx, dg = torch.autograd.grad(gated_linear_recurrence(x, g), [x, g], do)
    f = lambda xx, gg: float((oracle(xx, gg, None, None)[0]["o"] * do.double().cpu()).sum())
    xd, gd, h = x.detach().double(), g.detach().double(), 1e-6
    for t, d in ((0, 0), (17, 1), (39, 0)):
        e = torch.zeros_like(xd)
        e[0, t, d] = h
        # the loss is linear in x and smooth in g: differences of 64-bit values err by 1e-9,
        # fp32 gradients of magnitude 30 by 16 u 40 of it
        assert abs((f(xd + e, gd) - f(xd - e, gd)) / (2 * h) - float(dx[0, t, d])) < 2e-3
        assert abs((f(xd, gd + e) - f(xd, gd - e)) / (2 * h) - float(dg[0, t, d])) < 2e-3
