"""layer_norm against the formula in 64 bits: values, the residual's sum, gradients.

Tolerances count roundings, u = 2^-24 the half step of fp32: a row's sums of n terms err by
at most n u of the sum of magnitudes (blocked sums by less), the norm's few products by a
few u of what they multiply; then the result's own half step.
"""
import pytest
import torch

from hattention.norm_apis import layer_norm

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
BF, FH, FS = torch.bfloat16, torch.float16, torch.float32


def half(t):
    return torch.finfo(t).eps / 2


def make(seed, *shape, dtype=FS, scale=1.0, shift=0.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * scale + shift).to(dtype).to(DEV)


def oracle(x, weight, bias, residual, eps, dy=None, ds=None):
    """(results, bounds) in 64 bits."""
    f = lambda t: t.double() if t is not None else None
    n = x.shape[-1]
    s = x if residual is None else (x.float() + residual.float()).to(residual.dtype)
    sd = f(s)
    w = f(weight) if weight is not None else torch.ones(n, dtype=torch.float64, device=DEV)
    b = f(bias) if bias is not None else torch.zeros(n, dtype=torch.float64, device=DEV)
    mean = sd.mean(-1, keepdim=True)
    c = sd - mean
    rstd = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    hat = c * rstd
    # a centred value errs by the mean's error and a half step, a hat by that and by rstd's
    # relative error, which is half the variance's: sums of at most 64 terms a lane, then
    # of lanes (10 more steps), so 80 u
    dhat = 80 * U * (sd.abs().mean(-1, keepdim=True) + sd.abs()) * rstd + 80 * U * hat.abs()
    out = {"y": hat * w + b}
    tol = {"y": dhat * w.abs() + 4 * U * (hat.abs() * w.abs() + b.abs())}
    if residual is not None:
        out["s"], tol["s"] = sd, torch.zeros_like(sd)
    if dy is not None:
        dyd = f(dy)
        t = dyd * w
        m1, m2 = t.mean(-1, keepdim=True), (t * hat).mean(-1, keepdim=True)
        dx = rstd * (t - m1 - hat * m2)
        e = 160 * U * rstd * (t.abs() + t.abs().mean(-1, keepdim=True)
                              + hat.abs() * (t * hat).abs().mean(-1, keepdim=True))
        e = e + rstd * (dhat * m2.abs() + hat.abs() * (t.abs() * dhat).mean(-1, keepdim=True))
        if ds is not None:
            dx = dx + f(ds)
            e = e + 2 * U * f(ds).abs()
        rows = dyd.reshape(-1, n).shape[0]
        sums = (rows / 512 + 600) * U  # a wave's rows in turn, at most 512 partial rows
        flat = lambda z: z.reshape(-1, n)
        out.update(dx=dx, dweight=flat(dyd * hat).sum(0), dbias=flat(dyd).sum(0))
        tol.update(dx=e, dweight=flat((dyd * hat).abs()).sum(0) * sums
                   + flat(dyd.abs() * dhat).sum(0), dbias=flat(dyd.abs()).sum(0) * sums)
    return out, tol


def close(name, got, want, tol):
    d = (got.double() - want).abs()
    lim = tol + half(got.dtype) * (want.abs() + tol) + torch.finfo(got.dtype).smallest_normal
    bad = ~(d <= lim)
    assert not bad.any(), (name, float(d.max()), float((d / lim).max()))


CASES = [  # rows, n, x, parameters, residual
    (1, 1, FS, FS, None), (1, 16, BF, BF, BF), (3, 63, FH, FS, FH), (5, 1000, BF, FS, FS),
    (64, 1024, BF, BF, BF), (1025, 1024, BF, FS, BF), (2050, 512, FH, FH, FS),
    (1030, 2048, FS, FS, FS), (1026, 1531, BF, BF, None), (7, 2304, FS, FS, None),
    (9, 4097, FS, FS, FS), (3, 8192, BF, FS, BF), (2, 16384, FH, FS, None), (2, 16381, FS, FS, None),
    (4100, 64, BF, BF, FS), (1, 8, FS, BF, FS),
]


@pytest.mark.parametrize("rows,n,xt,pt,rt", CASES)
def test_forward_and_gradients(rows, n, xt, pt, rt):
    x = make(1, rows, n, dtype=xt, scale=2.0, shift=0.5).requires_grad_()
    w = make(2, n, dtype=pt, scale=0.3, shift=1.0).requires_grad_()
    b = make(3, n, dtype=pt, scale=0.5).requires_grad_()
    r = make(4, rows, n, dtype=rt, scale=3.0).requires_grad_() if rt else None
    dy = make(5, rows, n, dtype=xt)
    ds = make(6, rows, n, dtype=rt) if rt else None
    out = layer_norm(x, w, b, residual=r, eps=1e-5)
    y, s = out if rt else (out, None)
    leaves = [x, w, b] + ([r] if rt else [])
    g = torch.autograd.grad([y] + ([s] if rt else []), leaves, [dy] + ([ds] if rt else []))
    want, tol = oracle(x.detach(), w.detach(), b.detach(), r.detach() if rt else None, 1e-5, dy, ds)
    close("y", y, want["y"], tol["y"])
    close("dx", g[0], want["dx"], tol["dx"])
    close("dweight", g[1], want["dweight"], tol["dweight"])
    close("dbias", g[2], want["dbias"], tol["dbias"])
    if rt:
        assert torch.equal(s.double(), want["s"])
        close("dresidual", g[3], want["dx"], tol["dx"])
    # without gradients: the same values
    with torch.no_grad():
        again = layer_norm(x, w, b, residual=r, eps=1e-5)
    assert torch.equal(again[0] if rt else again, y)


@pytest.mark.parametrize("which", ["weight", "bias", "none"])
def test_missing_parameters(which):
    x = make(1, 37, 200, dtype=BF).requires_grad_()
    w = make(2, 200, shift=1.0).requires_grad_() if which == "weight" else None
    b = make(3, 200).requires_grad_() if which == "bias" else None
    dy = make(5, 37, 200, dtype=BF)
    y = layer_norm(x, w, b)
    leaves = [t for t in (x, w, b) if t is not None]
    g = torch.autograd.grad(y, leaves, dy)
    want, tol = oracle(x.detach(), w, b, None, 1e-5, dy)
    close("y", y, want["y"], tol["y"])
    close("dx", g[0], want["dx"], tol["dx"])
    if which != "none":
        close("dp", g[1], want["d" + which], tol["d" + which])


def test_only_some_gradients():
    x, r = make(1, 9, 64, dtype=BF), make(2, 9, 64, dtype=FS)
    w = make(3, 64).requires_grad_()
    y, s = layer_norm(x, w, None, residual=r)
    assert not torch.is_grad_enabled() or y.requires_grad
    (gw,) = torch.autograd.grad(y, [w], torch.ones_like(y))
    want, tol = oracle(x, w.detach(), None, r, 1e-5, torch.ones_like(y))
    close("dweight", gw, want["dweight"], tol["dweight"])
    # only the sum is used: its gradient passes through
    r2 = r.clone().requires_grad_()
    _, s = layer_norm(x, None, None, residual=r2)
    (gr,) = torch.autograd.grad(s, [r2], torch.full_like(s, 3.0))
    assert torch.equal(gr, torch.full_like(s, 3.0))


def test_views_and_offsets():
    """Rows that do not start on 16 bytes, transposed and expanded tensors."""
    base = make(1, 13 * 64 + 3, dtype=BF)
    x = base[3:].view(13, 64)
    w = make(2, 128)[::2]
    dy = make(3, 64, 13, dtype=BF).t()
    xg = x.detach().requires_grad_()
    y = layer_norm(xg, w)
    (g,) = torch.autograd.grad(y, [xg], dy)
    want, tol = oracle(x, w, None, None, 1e-5, dy)
    close("y", y, want["y"], tol["y"])
    close("dx", g, want["dx"], tol["dx"])
    y3 = layer_norm(x.view(13, 1, 64).expand(13, 2, 64), w)
    assert torch.equal(y3[:, 0], y) and torch.equal(y3[:, 1], y)


def test_large_offset_and_empty():
    """A mean far above the spread: the centred sum keeps it."""
    x = make(1, 4, 1024, shift=1000.0)
    want, _ = oracle(x, None, None, None, 1e-5)
    # x carries a half step of 1000 (3e-5) into a spread of 1; the mean as much again
    assert (layer_norm(x).double() - want["y"]).abs().max() < 2 * 1000 * 80 * U
    e = torch.empty(0, 64, device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    y = layer_norm(e, w)
    gx, gw = torch.autograd.grad(y, [e, w], torch.empty(0, 64, device=DEV))
    assert y.shape == (0, 64) and gx.shape == (0, 64) and torch.equal(gw, torch.zeros_like(w))


def test_nan_stays_in_its_row():
    x = make(1, 6, 96)
    x[2, 5] = float("nan")
    x[4, 7] = float("inf")
    y = layer_norm(x)
    assert y[2].isnan().all() and y[4].isnan().all()
    rows = [0, 1, 3, 5]
    want, tol = oracle(x[rows], None, None, None, 1e-5)
    close("y", y[rows], want["y"], tol["y"])


def test_difference_quotient():
    """The gradient against central differences of the formula in 64 bits."""
    x = make(1, 2, 24).requires_grad_()
    w = make(2, 24, shift=1.0)
    dy = make(3, 2, 24)
    (g,) = torch.autograd.grad(layer_norm(x, w), [x], dy)
    xd, h = x.detach().double(), 1e-6

    def loss(z):
        c = z - z.mean(-1, keepdim=True)
        return (c / (c.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w.double() * dy.double()).sum()
    for i, j in ((0, 0), (0, 13), (1, 23)):
        e = torch.zeros_like(xd)
        e[i, j] = h
        q = (loss(xd + e) - loss(xd - e)) / (2 * h)
        # h^2 of the third derivative and 2^-52 / h of the values: below 1e-7; fp32 below 1e-5
        assert abs(q - g[i, j].double()) < 2e-5
