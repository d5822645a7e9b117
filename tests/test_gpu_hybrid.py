"""The hybrid stack's mixers and norm as they are used: together, while decoding, captured
into graphs, on other streams, and on tensors whose offsets pass 32 bits."""
import pytest
import torch

from hattention.norm_apis import layer_norm
from hattention.recurrence_apis import gated_linear_recurrence, gated_linear_recurrence_step
from hattention.sliding_apis import (SlidingState, sliding_window_attention,
                                     sliding_window_prefill, sliding_window_step)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FS = torch.bfloat16, torch.float32
B, H, G, D, W, S = 2, 4, 2, 64, 50, 4
N = H * D


def make(seed, *shape, dtype=BF, scale=1.0, shift=0.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * scale + shift).to(dtype).to(DEV)


def parameters():
    p = {"w1": make(11, N, dtype=FS, scale=0.1, shift=1.0), "b1": make(12, N, dtype=FS, scale=0.1),
         "w2": make(13, N, dtype=FS, scale=0.1, shift=1.0), "b2": make(14, N, dtype=FS, scale=0.1)}
    p["gate"] = make(15, N, N, scale=N ** -0.5)
    p["qkv"] = make(16, N, (H + 2 * G) * D, scale=N ** -0.5)
    p["out"] = make(17, N, N, scale=N ** -0.5)
    return p


def decays(z):
    return -torch.nn.functional.softplus(z.float())


def block(x, p, lengths=None, cache=None):
    """norm -> recurrence -> norm with the residual stream -> attention; cache: filled with
    what decoding goes on from."""
    u = layer_norm(x, p["w1"], p["b1"])
    r = gated_linear_recurrence(u, decays(u @ p["gate"]), None, cache is not None, lengths)
    if cache is not None:
        r, cache["h"] = r
    y, s = layer_norm(r, p["w2"], p["b2"], residual=x)
    q, k, v = (t.unflatten(-1, (-1, D)) for t in (y @ p["qkv"]).split([H * D, G * D, G * D], -1))
    if cache is not None:
        o, cache["kv"] = sliding_window_prefill(q, k, v, W, S, lengths=lengths)
    else:
        o = sliding_window_attention(q, k, v, W, S, lengths=lengths)
    return s + o.flatten(-2) @ p["out"]


def token(x, p, cache):
    u = layer_norm(x, p["w1"], p["b1"])
    r, _ = gated_linear_recurrence_step(cache["h"], u, decays(u @ p["gate"]))
    y, s = layer_norm(r, p["w2"], p["b2"], residual=x)
    q, k, v = (t.unflatten(-1, (-1, D)) for t in (y @ p["qkv"]).split([H * D, G * D, G * D], -1))
    o, _ = sliding_window_step(cache["kv"], q, k, v)
    return s + o.flatten(-2) @ p["out"]


def oracle(x, p):
    """The same block in 64 bits, by elementary operations."""
    def norm(z, w, b):
        c = z - z.mean(-1, keepdim=True)
        return c / (c.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w + b
    T = x.shape[1]
    u = norm(x, p["w1"], p["b1"])
    a, h, hs = torch.exp(-torch.nn.functional.softplus(u @ p["gate"])), 0.0, []
    for t in range(T):
        h = a[:, t] * h + u[:, t]
        hs.append(h)
    s = x + torch.stack(hs, 1)
    y = norm(s, p["w2"], p["b2"])
    q, k, v = (t.unflatten(-1, (-1, D)).transpose(1, 2)
               for t in (y @ p["qkv"]).split([H * D, G * D, G * D], -1))
    k, v = (t.repeat_interleave(H // G, 1) for t in (k, v))
    i = torch.arange(T, device=x.device)
    gone = (i > i[:, None]) | ((i[:, None] - i >= W) & (i >= S))
    z = (q @ k.transpose(-1, -2).contiguous() * D ** -0.5).masked_fill(gone, -torch.inf)
    o = (torch.softmax(z, -1) @ v).transpose(1, 2).flatten(-2)
    return s + o @ p["out"]


def apart(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


# A pass of the block rounds to bf16 at most 12 times one after the other (u, the gate's
# product, its decay's argument, r, s, y, qkv, P, o, its product, the sum, the result), each by
# a relative half step 2^-8 of what it passes on; a norm and a softmax hand errors on about as
# large as they came in.  A gradient goes back through as many and was computed from them.
FORWARD, BACKWARD = 12 * 2.0 ** -8, 24 * 2.0 ** -8


@pytest.mark.parametrize("T", [1, 37, 300])
def test_training_together(T):
    x, p = make(1, B, T, N).requires_grad_(), parameters()
    leaves = [x] + [t.requires_grad_() for t in p.values()]
    do = make(2, B, T, N)
    y = block(x, p)
    grads = torch.autograd.grad(y, leaves, do)
    x64 = x.detach().double().requires_grad_()
    p64 = {n: t.detach().double().requires_grad_() for n, t in p.items()}
    want = oracle(x64, p64)
    ref = torch.autograd.grad(want, [x64, *p64.values()], do.double())
    assert apart(y.detach(), want.detach()) < FORWARD
    for n, a, b in zip(["x", *p], grads, ref):
        # at T = 1 each query sees one key and the gate meets no state: those are zero
        if float(b.norm()) == 0:
            assert not a.any(), n
        else:
            assert apart(a, b) < BACKWARD, (n, apart(a, b))


def test_decoding_together():
    """A padded batch of prompts, then tokens: each row as one sequence of its own."""
    p, new, lens = parameters(), 9, [70, 33]
    full = [make(20 + b, 1, n + new, N) for b, n in enumerate(lens)]
    x = torch.full((B, max(lens), N), float("nan"), device=DEV, dtype=BF)
    for b, n in enumerate(lens):
        x[b, :n] = full[b][0, :n]
    # the norms read padded rows too, so padding is finite there
    x = torch.where(x.isnan(), torch.zeros_like(x), x)
    cache, lengths = {}, torch.tensor(lens, device=DEV)
    with torch.no_grad():
        prompt = block(x, p, lengths, cache)
        steps = [token(torch.cat([full[b][:, n + i] for b, n in enumerate(lens)]), p, cache)
                 for i in range(new)]
    p64 = {n: t.double() for n, t in p.items()}
    for b, n in enumerate(lens):
        want = oracle(full[b].double(), p64)[0]
        assert apart(prompt[b, :n], want[:n]) < FORWARD
        assert apart(torch.stack([s[b] for s in steps]), want[n:]) < FORWARD


def capture(fn):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            fn()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return graph, out


def test_captured_training():
    """A captured forward and backward, replayed on new inputs between eager passes."""
    T, p = 600, parameters()
    x, do = make(1, B, T, N).requires_grad_(), make(2, B, T, N)
    leaves = [x] + [t.requires_grad_() for t in p.values()]

    def step():
        y = block(x, p)
        return [y.detach(), *torch.autograd.grad(y, leaves, do)]
    graph, out = capture(step)
    for seed in range(3):
        with torch.no_grad():
            x.copy_(make(30 + seed, B, T, N))
            do.copy_(make(40 + seed, B, T, N))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        eager = step()
        torch.cuda.synchronize()
        for a, b in zip(got, eager):
            assert torch.equal(a, b)


def test_captured_steps():
    """A captured token step advances its state with each replay; two captures of one
    function keep apart."""
    p = parameters()

    def fresh():
        return {"h": torch.zeros(B, N, device=DEV),
                "kv": SlidingState.empty(B, G, D, W, S, device=DEV)}
    x = make(1, B, N)
    caches, eager = [fresh(), fresh()], fresh()
    graphs = []
    with torch.no_grad():
        for c in caches:
            saved = {"h": c["h"].clone()}
            graphs.append(capture(lambda: token(x, p, c)))
            c["h"].copy_(saved["h"])
            for t in (c["kv"].k, c["kv"].v, c["kv"].counts):
                t.zero_()
        for i in range(70):
            x.copy_(make(50 + i, B, N))
            want = token(x, p, eager)
            for graph, out in graphs:
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(out, want), i
    for c in caches:
        assert torch.equal(c["h"], eager["h"]) and torch.equal(c["kv"].k, eager["kv"].k)
        assert c["kv"].counts.tolist() == [70] * B


def test_other_streams_at_once():
    """Calls that overlap on two streams, each with its own workspaces."""
    T, p = 700, parameters()
    xs = [make(60 + i, B, T, N).requires_grad_() for i in range(2)]
    do = make(2, B, T, N)

    def step(x):
        y = block(x, p)
        return [y.detach(), *torch.autograd.grad(y, [x], do)]
    want = [step(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for x, s in zip(xs, streams):
            with torch.cuda.stream(s):
                got.append(step(x))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


# ------------------------------------------------------------- offsets past 32 bits
def test_large_norm_and_recurrence():
    n, rows = 4096, 2 ** 19 + 3  # 2^31 elements and more
    x = torch.zeros(rows, n, device=DEV, dtype=BF)
    x[-5:] = make(1, 5, n)
    w = make(2, n, dtype=FS, shift=1.0)
    y = layer_norm(x, w)
    assert torch.equal(y[-5:], layer_norm(x[-5:].clone(), w))
    del y
    xg = x.requires_grad_()
    (g,) = torch.autograd.grad(layer_norm(xg, w), [xg], xg.detach())
    tail = x.detach()[-5:].clone().requires_grad_()
    (want,) = torch.autograd.grad(layer_norm(tail, w), [tail], tail.detach())
    # other numbers of rows take other kernels: equal to fp32's rounding, then to bf16's
    assert (g[-5:].double() - want.double()).abs().max() <= 2.0 ** -8 * want.abs().max()
    del g, xg
    z = x.detach().view(1, rows, n)
    decay = torch.full((1, 1, 1), -1.0, device=DEV, dtype=BF).expand(z.shape).contiguous()
    h = gated_linear_recurrence(z, decay)
    tail = gated_linear_recurrence(z[:, -5:].contiguous(), decay[:, -5:].contiguous())
    assert torch.equal(h[:, -5:], tail)


def test_large_attention():
    T, H_, D_ = 2 ** 17 + 70, 128, 128
    q = torch.zeros(1, T, H_, D_, device=DEV, dtype=BF)
    q[:, -300:] = make(1, 1, 300, H_, D_)
    k, v = make(2, 1, T, 1, D_), make(3, 1, T, 1, D_)
    q.requires_grad_()
    o = sliding_window_attention(q, k, v, 100)
    (dq,) = torch.autograd.grad(o, [q], q.detach())
    cut = 128 * (T // 128 - 2)  # a tail that begins a block of queries, with its window
    qt = q.detach()[:, cut:].clone().requires_grad_()
    ot = sliding_window_attention(qt, k[:, cut:], v[:, cut:], 100)
    (dt,) = torch.autograd.grad(ot, [qt], qt.detach())
    # past the tail's first window the two see the same keys, in other tiles: P's rounding, and
    # the result's
    lim = 2.0 ** -7 * v.abs().max()
    assert (o[:, cut + 128:].double() - ot[:, 128:].double()).abs().max() < lim
    assert apart(dq[:, cut + 128:], dt[:, 128:]) < 6 * 2.0 ** -8


def test_large_cache():
    B_, G_, D_, W_ = 65, 8, 128, 2 ** 15
    state = SlidingState.empty(B_, G_, D_, W_, device=DEV)  # 2^31 elements and more
    small = SlidingState.empty(1, G_, D_, 300, device=DEV)
    state.counts[-1] = 200
    small.counts[0] = 200
    rows = make(1, G_, 200, D_)
    for s in (state, small):
        s.k[-1, :, :200] = rows
        s.v[-1, :, :200] = rows
    q, k, v = make(2, B_, G_, D_), make(3, B_, G_, D_), make(4, B_, G_, D_)
    o, _ = sliding_window_step(state, q, k, v)
    want, _ = sliding_window_step(small, q[-1:], k[-1:], v[-1:])
    # the splits differ with the window: P's rounding, and the result's
    assert (o[-1].double() - want[0].double()).abs().max() < 2.0 ** -7 * rows.abs().max()
    assert torch.equal(state.k[-1, :, 200], k[-1]) and torch.equal(o[0], v[0])
