"""Sliding-window attention against 64 bits by the norm of the error.

A bound on each element adds up worst cases, and over thousands of queries becomes as large as the
gradients.  Roundings are independent, so the error's square adds up their variances instead.  A
rounding to a type of half step h (relative) has a variance of at most (h x)^2 / 3, and:
* o = P V: P is rounded, and o;
* dV = P^T dO: P is rounded, and dV;
* delta = rowsum(dO o) is taken from the rounded o: its variance is (h^2 / 3) times
  sum (P dP)^2 + sum (dO o)^2 over the row;
* dS = P (dP - delta) is rounded, and carries P times delta's error, in dQ through K (one error for
  all keys of a row: (P K)^2), in dK through Q; dQ and dK are rounded.
32-bit products and sums (2^-24 each) do not count beside h.  The variance of a rounding is 0.54 of
the bound where mantissas are spread evenly over a binade's logarithm, and the squared norms below
add at least a hundred independent terms: 1.5 times the bound is met by all right results.
That it sees mistakes is tested on the CPU.
"""
import math

import pytest
import torch

from hattention.sliding_apis import sliding_window_attention

BF, FH = torch.bfloat16, torch.float16
NAMES = ("o", "dq", "dk", "dv")


def inputs(B, T, H, G, D, dtype):
    def make(seed, n):
        return torch.randn(B, T, n, D, generator=torch.Generator().manual_seed(seed)).to(dtype)
    return make(1, H), make(2, G), make(3, G), make(4, H)


def rounded(x, dtype):
    return x if dtype is None else x.to(dtype).to(x.dtype)


def formula(q, k, v, do, W, S, lengths=None, scale=None, to=None, wrong=None):
    """({name: result}, {name: bound of the error's variance}) in 64 bits.  `to`: P, dS and the
    results are rounded to that type, as the kernels round them; `wrong` plants a mistake in dK
    and dV (that of delta reaches dQ too)."""
    B, T, H, D = q.shape
    G, dev = k.shape[2], q.device
    R, scale = H // G, D ** -0.5 if scale is None else scale
    var = (torch.finfo(q.dtype).eps / 2) ** 2 / 3
    z = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=dev)
    out = {n: z(t) for n, t in zip(NAMES, (q, q, k, v))}
    err = {n: z(t) for n, t in out.items()}
    i = torch.arange(T, device=dev)
    seen = (i <= i[:, None]) & ((i[:, None] - i < W) | (i < S))
    for b in range(B):
        n = T if lengths is None else lengths[b]
        for h in range(H):
            g, m = h // R, seen[:n, :n]
            qi, ki, vi, gi = (t[b, :n, j].double() for t, j in ((q, h), (k, g), (v, g), (do, h)))
            p = torch.softmax((qi @ ki.T * scale).masked_fill(~m, -math.inf), 1)
            dp = (gi @ vi.T).masked_fill(~m, 0)
            o = rounded(rounded(p, to) @ vi, to)
            delta = (gi * o).sum(1, keepdim=True) if to else (p * dp).sum(1, keepdim=True)
            if wrong == "delta":
                delta = delta * 0.9
            ds = p * (dp - delta)
            pr, dr = rounded(p, to), rounded(ds, to)
            dq = dr @ ki * scale
            if wrong == "one chunk of one head's far queries" and h == 0:
                # the sinks without the last chunk of 1024 queries past the window
                last = W + (n - W - 1) // 1024 * 1024
                far = (i[:n, None] >= last) & (i[:n] < S) & (i[:n, None] - i[:n] >= W)
                pr, dr = pr.masked_fill(far, 0), dr.masked_fill(far, 0)
            if wrong == "a tile of 32 queries" and h == 0:
                pr, dr = pr.clone(), dr.clone()
                pr[256:288], dr[256:288] = 0, 0
            if wrong == "a tile of 32 keys" and h == 0:
                pr, dr = pr.clone(), dr.clone()
                pr[:, 256:288], dr[:, 256:288] = 0, 0
            if wrong == "the last query of a key's window" and h == 0:
                edge = (i[:n, None] - i[:n] == W - 1) & (i[:n] < 128)
                pr, dr = pr.masked_fill(edge, 0), dr.masked_fill(edge, 0)
            own = h != H - 1 if wrong == "one head" else True
            sd = var * ((p * dp).square().sum(1) + (gi * o).square().sum(1))[:, None]
            out["o"][b, :n, h], out["dq"][b, :n, h] = o, dq
            err["o"][b, :n, h] = var * (p.square() @ vi.square() + o.square())
            err["dq"][b, :n, h] = scale ** 2 * (var * ds.square() @ ki.square()
                                                + sd * (p @ ki).square())
            if own:
                out["dk"][b, :n, g] += dr.T @ qi * scale
                out["dv"][b, :n, g] += pr.T @ gi
            err["dk"][b, :n, g] += scale ** 2 * ((var * ds.square() + sd * p.square()).T @ qi.square())
            err["dv"][b, :n, g] += var * p.square().T @ gi.square()
    for n in NAMES[1:]:
        err[n] += var * out[n].square()
    return {n: rounded(t, to) for n, t in out.items()}, err


def ratios(got, want, err, S, lengths=None):
    """{part: |error|^2 / its bound}: each tensor whole, its rows of each batch in blocks of 128 (a
    last one of up to 255), and the sinks of dk and dv."""
    r = {}
    for n in NAMES:
        d = (got[n].double() - want[n]).square()
        r[n] = float(d.sum() / err[n].sum())
        for b in range(d.shape[0]):
            end = d.shape[1] if lengths is None else lengths[b]
            cuts = list(range(0, max(end - 127, 1), 128)) + [end]
            for lo, hi in zip(cuts, cuts[1:]):
                r[n, b, lo] = float(d[b, lo:hi].sum() / err[n][b, lo:hi].sum())
            if S and n in ("dk", "dv"):
                m = min(S, end)
                r[n, b, "sinks"] = float(d[b, :m].sum() / err[n][b, :m].sum())
    return r


LIMIT = 1.5
CASES = [  # B, T, H, G, D, W, S, dtype, lengths, scale
    (1, 2500, 4, 2, 64, 200, 40, BF, None, None), (1, 1300, 2, 1, 64, 65, 4, BF, None, None),
    (1, 4500, 2, 1, 128, 3000, 16, BF, None, 0.3), (1, 2500, 4, 1, 128, 100, 33, FH, None, None),
    (2, 2400, 2, 2, 64, 130, 8, BF, [2400, 1500], None), (1, 2200, 2, 2, 80, 70, 64, FH, None, None),
    (1, 700, 2, 1, 64, 20, 3, BF, None, None), (1, 1500, 3, 1, 96, 600, 0, BF, None, None),
    (1, 3200, 8, 1, 64, 64, 2, BF, None, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,H,G,D,W,S,dtype,lens,scale", CASES)
def test_error_norms(B, T, H, G, D, W, S, dtype, lens, scale):
    q, k, v, do = (t.to("cuda:0") for t in inputs(B, T, H, G, D, dtype))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    n = torch.tensor(lens, dtype=torch.int32, device="cuda:0") if lens else None
    o = sliding_window_attention(*leaves, W, S, scale, n)
    grads = torch.autograd.grad(o, leaves, do)
    got = dict(zip(NAMES, (o.detach(), *grads)))
    want, err = formula(q.detach(), k.detach(), v.detach(), do, W, S, lens, scale)
    r = ratios(got, want, err, S, lens)
    worst = max(r, key=lambda p: r[p])
    print({n: round(r[n], 2) for n in NAMES}, worst, round(r[worst], 2))
    assert r[worst] < LIMIT, (worst, r[worst], {n: r[n] for n in NAMES})


WRONG = ["delta", "one chunk of one head's far queries", "a tile of 32 queries",
         "a tile of 32 keys", "the last query of a key's window", "one head"]


@pytest.mark.parametrize("B,T,H,G,D,W,S,dtype", [(1, 2500, 4, 2, 64, 200, 40, BF),
                                                 (1, 1300, 2, 1, 64, 65, 4, BF)])
def test_the_limit_tells_roundings_from_mistakes(B, T, H, G, D, W, S, dtype):
    ins = inputs(B, T, H, G, D, dtype)
    want, err = formula(*ins, W, S)
    right = ratios(formula(*ins, W, S, to=dtype)[0], want, err, S)
    assert max(right.values()) < LIMIT, max(right.items(), key=lambda p: p[1])
    for wrong in WRONG:
        r = ratios(formula(*ins, W, S, to=dtype, wrong=wrong)[0], want, err, S)
        for n in ("dk",) if wrong == "delta" else ("dk", "dv"):
            top = max((x, part) for part, x in r.items() if n in part)
            print(wrong, n, top, r.get((n, 0, "sinks")))
            assert top[0] > 2 * LIMIT, (wrong, n, top)
