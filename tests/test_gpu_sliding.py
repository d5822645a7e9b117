"""Sliding-window attention with sinks against the formula in 64 bits.

Tolerances count roundings.  With h the half step of the inputs' dtype and u = 2^-24:
* a probability is rounded to that dtype, P (1 + h), and carries the errors of its score
  (D products in fp32, |s| (D + 4) u each) and of the sum: r = h + 2 (D + 8) u max|s| + T u;
* o = P V errs by r sum P |v|, then by its own half step;
* dS = P (dP - delta): delta is taken from the rounded o, so it errs by sum |do| d_o, where
  d_o is o's bound; dS is rounded: h |dS|; both enter dQ and dK through sums of magnitudes;
* every sum adds its length in u of its magnitudes.
"""
import math

import pytest
import torch

from hattention.sliding_apis import (SlidingState, sliding_window_attention,
                                     sliding_window_prefill, sliding_window_step)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
BF, FH = torch.bfloat16, torch.float16


def make(seed, *shape, dtype=BF, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * scale).to(dtype).to(DEV)


def seen(T, W, S):
    t, s = torch.arange(T, device=DEV)[:, None], torch.arange(T, device=DEV)
    return (s <= t) & ((t - s < W) | (s < S))


def oracle(q, k, v, W, S, scale=None, lengths=None, do=None):
    """(results, bounds) in 64 bits on the device."""
    B, T, H, D = q.shape
    G = k.shape[2]
    R = H // G
    h = torch.finfo(q.dtype).eps / 2
    scale = D ** -0.5 if scale is None else scale
    z = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=DEV)
    out = {"o": z(q), "dq": z(q), "dk": z(k), "dv": z(v)}
    tol = {n: z(t) for n, t in out.items()}
    for b in range(B):
        n = T if lengths is None else min(max(int(lengths[b]), 0), T)
        if n == 0:
            continue
        m = seen(n, W, S)
        for i in range(H):
            g = i // R
            qi, ki, vi = q[b, :n, i].double(), k[b, :n, g].double(), v[b, :n, g].double()
            s = qi @ ki.T * scale
            p = torch.softmax(s.masked_fill(~m, -math.inf), 1)
            big = (qi.abs() @ ki.T.abs() * scale).masked_fill(~m, 0).amax()
            r = h + 2 * (D + 8) * U * big + n * U
            out["o"][b, :n, i] = p @ vi
            do_ = r * (p @ vi.abs())
            tol["o"][b, :n, i] = do_
            if do is None:
                continue
            gi = do[b, :n, i].double()
            dp = (gi @ vi.T).masked_fill(~m, 0)
            ds = p * (dp - (p * dp).sum(1, keepdim=True))
            o_err = do_ + h * (p @ vi).abs()
            mag = (gi.abs() @ vi.T.abs()).masked_fill(~m, 0)  # what dp sums
            e_ds = p * ((gi.abs() * o_err).sum(1, keepdim=True) + (2 * D + n) * U
                        * (mag + (p * mag).sum(1, keepdim=True))) + r * ds.abs()
            out["dq"][b, :n, i] = ds @ ki * scale
            tol["dq"][b, :n, i] = (e_ds + n * U * ds.abs()) @ ki.abs() * scale
            out["dk"][b, :n, g] += ds.T @ qi * scale
            tol["dk"][b, :n, g] += (e_ds + R * n * U * ds.abs()).T @ qi.abs() * scale
            out["dv"][b, :n, g] += p.T @ gi
            tol["dv"][b, :n, g] += (r + R * n * U) * (p.T @ gi.abs())
    return out, tol


def close(name, got, want, tol):
    d = (got.double() - want).abs()
    f = torch.finfo(got.dtype)
    lim = tol + f.eps / 2 * (want.abs() + tol) + f.smallest_normal * f.eps
    bad = ~(d <= lim)
    assert not bad.any(), (name, float(d.max()), float((d / lim).max()), bad.nonzero()[:4].tolist())


CASES = [  # B, T, H, G, D, W, S, dtype, lengths
    (1, 1, 1, 1, 64, 1, 0, BF, None), (2, 2, 2, 1, 64, 5, 1, BF, None),
    (1, 33, 3, 3, 64, 8, 3, FH, None), (1, 64, 4, 2, 128, 64, 0, BF, None),
    (2, 130, 2, 2, 128, 1, 0, BF, None), (1, 129, 2, 1, 64, 1, 1, BF, None),
    (2, 200, 4, 1, 128, 31, 4, FH, [200, 77]), (1, 300, 2, 2, 64, 300, 64, BF, None),
    (1, 300, 2, 2, 64, 299, 64, BF, None), (3, 257, 6, 3, 80, 100, 16, BF, [257, 0, 1]),
    (1, 700, 2, 1, 96, 128, 33, FH, None), (1, 520, 8, 1, 8, 63, 5, BF, None),
    (2, 384, 2, 2, 128, 127, 64, BF, [384, 129]), (1, 1300, 2, 1, 64, 65, 4, BF, None),
    (1, 2500, 4, 2, 64, 200, 40, BF, [2300]), (1, 640, 20, 1, 64, 500, 2, FH, None),
    (1, 513, 1, 1, 120, 2 ** 30, 0, BF, None), (2, 190, 2, 2, 40, 50, 64, FH, [10, 190]),
]


@pytest.mark.parametrize("B,T,H,G,D,W,S,dtype,lens", CASES)
def test_forward_and_gradients(B, T, H, G, D, W, S, dtype, lens):
    q = make(1, B, T, H, D, dtype=dtype).requires_grad_()
    k = make(2, B, T, G, D, dtype=dtype).requires_grad_()
    v = make(3, B, T, G, D, dtype=dtype).requires_grad_()
    do = make(4, B, T, H, D, dtype=dtype)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV) if lens else None
    o = sliding_window_attention(q, k, v, W, S, lengths=n)
    grads = torch.autograd.grad(o, [q, k, v], do)
    want, tol = oracle(q.detach(), k.detach(), v.detach(), W, S, None, lens, do)
    for name, got in zip(["o", "dq", "dk", "dv"], [o.detach(), *grads]):
        close(name, got, want[name], tol[name])
    with torch.no_grad():
        assert torch.equal(sliding_window_attention(q, k, v, W, S, lengths=n), o)


def test_long_window_and_scale():
    B, T, H, G, D, W, S = 1, 4500, 2, 1, 128, 3000, 16
    q, k, v = (make(i, B, T, n, D).requires_grad_() for i, n in ((1, H), (2, G), (3, G)))
    do = make(4, B, T, H, D)
    o = sliding_window_attention(q, k, v, W, S, scale=0.3)
    grads = torch.autograd.grad(o, [q, k, v], do)
    want, tol = oracle(q.detach(), k.detach(), v.detach(), W, S, 0.3, None, do)
    for name, got in zip(["o", "dq", "dk", "dv"], [o.detach(), *grads]):
        close(name, got, want[name], tol[name])


def test_peaked_scores():
    """Scores far apart: the running maximum grows tile after tile, and one key wins."""
    B, T, H, D = 1, 600, 1, 64
    q = torch.full((B, T, H, D), 1.0, device=DEV, dtype=BF)
    k = (torch.arange(T, device=DEV) / 4).view(1, T, 1, 1).expand(B, T, H, D).to(BF).contiguous()
    v = make(3, B, T, H, D)
    o = sliding_window_attention(q, k, v, 400, 4)
    want, tol = oracle(q, k, v, 400, 4)
    close("o", o, want["o"], tol["o"])
    o = sliding_window_attention(q, -k, v, 400, 4)
    want, tol = oracle(q, -k, v, 400, 4)
    close("o", o, want["o"], tol["o"])


def test_scores_far_below_zero():
    """The largest score of a row is far below anything that a softmax usually meets."""
    B, T, H, D = 1, 200, 1, 64
    q = torch.full((B, T, H, D), 2.0 ** 60, device=DEV, dtype=BF)
    k = torch.full((B, T, H, D), -2.0 ** 58, device=DEV, dtype=BF)
    v = make(3, B, T, H, D)
    want, tol = oracle(torch.zeros_like(q), k, v, 90, 4)  # equal scores: the keys' mean
    close("o", sliding_window_attention(q, k, v, 90, 4), want["o"], tol["o"])
    state = SlidingState.empty(B, H, D, 90, 4, device=DEV)
    for t in range(120):
        o, _ = sliding_window_step(state, q[:, t], k[:, t], v[:, t])
    close("step", o, want["o"][:, 119], tol["o"][:, 119])


def test_one_visible_key_has_no_score_gradient():
    q, k, v = (make(i, 1, 200, 2, 64).requires_grad_() for i in (1, 2, 3))
    o = sliding_window_attention(q, k, v, 1)
    dq, dk, dv = torch.autograd.grad(o, [q, k, v], make(4, 1, 200, 2, 64))
    wide = sliding_window_attention(q, k, v, 2 ** 40)  # any whole number is a window
    assert torch.equal(wide, sliding_window_attention(q, k, v, 200))
    assert torch.equal(o, v) and not dq.any() and not dk.any() and torch.equal(dv, make(4, 1, 200, 2, 64))


def test_views_are_read_in_place():
    """q, k, v as windows of one projection, transposed heads, expanded keys, odd offsets."""
    B, T, H, G, D = 2, 150, 4, 2, 64
    packed = make(1, B, T, (H + 2 * G) * D)
    q, k, v = (t.unflatten(-1, (-1, D)) for t in packed.split([H * D, G * D, G * D], -1))
    do = make(4, B, T, H, D)
    ref = [t.clone().requires_grad_() for t in (q, k, v)]
    want = sliding_window_attention(*ref, 40, 4)
    gw = torch.autograd.grad(want, ref, do)
    forms = {
        "windows": (q, k, v),
        "heads first": tuple(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)),
        "last dimension apart": tuple(t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v)),
        "odd offset": tuple(torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape)
                            for t in (q, k, v)),
    }
    for name, ts in forms.items():
        leaves = [t.detach().requires_grad_() for t in ts]
        o = sliding_window_attention(*leaves, 40, 4)
        assert torch.equal(o, want), name
        for a, b in zip(torch.autograd.grad(o, leaves, do.transpose(1, 2).contiguous().transpose(1, 2)), gw):
            assert torch.equal(a, b), name
    # one key head given to all heads by expand: its gradient is summed by autograd
    k1 = k[:, :, :1].detach().requires_grad_()
    o = sliding_window_attention(q, k1.expand(B, T, H, D), v[:, :, :1].expand(B, T, H, D), 40, 4)
    o2 = sliding_window_attention(q, k1, v[:, :, :1], 40, 4)
    # the head layouts may take different tiles, so they agree to the bound and not to the bit
    want, tol = oracle(q, k1.detach(), v[:, :, :1], 40, 4, None, None, do)
    close("o", o.detach(), want["o"], tol["o"])
    close("o2", o2.detach(), want["o"], tol["o"])
    (dk,) = torch.autograd.grad(o2, [k1], do)
    close("dk", dk, want["dk"], tol["dk"])
    (dk,) = torch.autograd.grad(o, [k1], do)
    # H gradients of their own, each rounded, added in bf16 (H - 1 more roundings)
    mine, each = oracle(q, k1.detach().expand(B, T, H, D), v[:, :, :1].expand(B, T, H, D), 40, 4,
                        None, None, do)
    mag = mine["dk"].abs().sum(2, keepdim=True)
    close("dk", dk, want["dk"], each["dk"].sum(2, keepdim=True) + H * 2.0 ** -8 * mag)


def test_padding_is_not_read():
    B, T, H, D = 2, 300, 2, 64
    q, k, v = (make(i, B, T, H, D) for i in (1, 2, 3))
    n = torch.tensor([300, 140], device=DEV)
    o = sliding_window_attention(q, k, v, 64, 4, lengths=n)
    bad = [t.clone() for t in (q, k, v)]
    for t in bad:
        t[1, 140:] = float("nan")
        t.requires_grad_()
    o2 = sliding_window_attention(*bad, 64, 4, lengths=n)
    assert torch.equal(o, o2) and not o2[1, 140:].any()
    do = make(4, B, T, H, D)
    do[1, 140:] = float("inf")
    for g in torch.autograd.grad(o2, bad, do):
        assert g.isfinite().all() and not g[1, 140:].any()


def test_nan_reaches_who_sees_it():
    B, T, H, D = 1, 500, 1, 64
    q, k, v = (make(i, B, T, H, D) for i in (1, 2, 3))
    v[0, 200, 0, 7] = float("nan")
    o = sliding_window_attention(q, k, v, 50)
    assert o[0, 200:250, 0, 7].isnan().all()
    assert o[0, :128].isfinite().all() and o[0, 384:].isfinite().all()


def test_same_bits_every_time():
    q, k, v = (make(i, 2, 1500, n, 64).requires_grad_() for i, n in ((1, 4), (2, 2), (3, 2)))
    do = make(4, 2, 1500, 4, 64)
    base = None
    for _ in range(3):
        o = sliding_window_attention(q, k, v, 300, 8)
        got = (o.detach(), *torch.autograd.grad(o, [q, k, v], do))
        base = base or got
        assert all(torch.equal(a, b) for a, b in zip(base, got))


def test_difference_quotient():
    B, T, H, D = 1, 70, 1, 64
    q, k, v = (make(i, B, T, H, D, dtype=FH).requires_grad_() for i in (1, 2, 3))
    do = make(4, B, T, H, D, dtype=FH)
    grads = torch.autograd.grad(sliding_window_attention(q, k, v, 20, 2), [q, k, v], do)
    leaves = [t.detach().double() for t in (q, k, v)]

    def loss(q, k, v):
        s = (q[0, :, 0] @ k[0, :, 0].T / 8).masked_fill(~seen(T, 20, 2), -math.inf)
        return float(((torch.softmax(s, 1) @ v[0, :, 0]) * do[0, :, 0].double()).sum())
    _, tol = oracle(q.detach(), k.detach(), v.detach(), 20, 2, None, None, do)
    for j, name in enumerate(("dq", "dk", "dv")):
        for t, d in ((0, 3), (30, 60), (69, 1)):
            e = torch.zeros_like(leaves[j])
            e[0, t, 0, d] = 1e-5
            p, m = list(leaves), list(leaves)
            p[j], m[j] = p[j] + e, m[j] - e
            want = (loss(*p) - loss(*m)) / 2e-5
            # the quotient errs by 1e-10 of the third derivative and 1e-15 / 1e-5 of the loss
            lim = float(tol[name][0, t, 0, d]) + 2.0 ** -11 * abs(want) + 1e-6
            assert abs(float(grads[j][0, t, 0, d]) - want) < lim, (name, t, d)


# ---------------------------------------------------------------------------- decode
STEPS = [  # B, H, G, D, W, S, dtype, prompt lengths
    (1, 1, 1, 64, 1, 0, BF, [1]), (2, 4, 2, 64, 8, 3, BF, [1, 30]), (3, 8, 1, 128, 40, 4, FH, [5, 44, 90]),
    (2, 34, 2, 128, 33, 0, BF, [33, 32]), (2, 6, 3, 80, 300, 16, BF, [10, 400]),
    (1, 16, 4, 64, 1000, 64, FH, [1100]), (4, 2, 2, 8, 5, 2, BF, [1, 2, 3, 40]),
]


@pytest.mark.parametrize("B,H,G,D,W,S,dtype,lens", STEPS)
def test_prefill_and_steps(B, H, G, D, W, S, dtype, lens):
    """A padded batch of prompts, then tokens one by one, against one long sequence."""
    T, new = max(lens), 12
    full = [make(i, B, T + new, n, D, dtype=dtype) for i, n in ((1, H), (2, G), (3, G))]
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    prompt = [t[:, :T].clone() for t in full]
    for b in range(B):
        for t in prompt:
            t[b, lens[b]:] = float("nan")
    o, state = sliding_window_prefill(*prompt, W, S, lengths=n)
    rows = torch.arange(B, device=DEV)
    got = []
    for i in range(new):
        # row b's token lens[b] + i of its own sequence
        q, k, v = (t[rows, (n + i).long()] for t in full)
        y, s = sliding_window_step(state, q, k, v)
        assert s is state
        got.append(y)
    assert state.counts.tolist() == [m + new for m in lens]
    for b in range(B):
        m = lens[b] + new
        one = [t[b:b + 1, :m] for t in full]
        want, tol = oracle(*one, W, S)
        close("prompt", o[b:b + 1, :lens[b]], want["o"][:, :lens[b]], tol["o"][:, :lens[b]])
        for i in range(new):
            close(f"step {i}", got[i][b], want["o"][0, lens[b] + i], tol["o"][0, lens[b] + i])
        # the cache holds the sinks and the last tokens, each in its slot
        for p in list(range(min(S, m))) + list(range(max(S, m - W), m)):
            slot = p if p < S else S + (p - S) % W
            assert torch.equal(state.k[b, :, slot], full[1][b, p])
            assert torch.equal(state.v[b, :, slot], full[2][b, p])


def test_steps_from_nothing_ignore_unwritten_slots():
    B, H, G, D, W, S = 2, 4, 2, 64, 100, 4
    state = SlidingState.empty(B, G, D, W, S, device=DEV)
    state.k.fill_(float("nan"))
    state.v.fill_(float("nan"))
    full = [make(i, B, 40, n, D) for i, n in ((1, H), (2, G), (3, G))]
    want, tol = oracle(*full, W, S)
    for t in range(40):
        o, _ = sliding_window_step(state, *(x[:, t] for x in full))
        close("o", o, want["o"][:, t], tol["o"][:, t])


def test_step_scale_and_views():
    B, H, G, D, W = 2, 4, 2, 64, 16
    kv = make(2, B, 2 * G, D)
    q = make(1, B, D, H).transpose(1, 2)
    outs = []
    for form in (lambda t: t, lambda t: t.contiguous()):
        state = SlidingState.empty(B, G, D, W, device=DEV)
        sliding_window_step(state, make(5, B, H, D), make(6, B, G, D), make(7, B, G, D))
        outs.append(sliding_window_step(state, form(q), form(kv[:, :G]), form(kv[:, G:]), scale=0.5)[0])
    assert torch.equal(*outs)
    full = [torch.stack([make(5, B, H, D), q], 1), torch.stack([make(6, B, G, D), kv[:, :G]], 1),
            torch.stack([make(7, B, G, D), kv[:, G:]], 1)]
    want, tol = oracle(*full, W, 0, 0.5)
    close("o", outs[0], want["o"][:, 1], tol["o"][:, 1])
