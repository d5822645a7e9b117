"""The global attention's operators as they are used: rotary positions, the cache and the
attention together, next to the sliding window, captured, on other streams and other devices."""
import functools

import pytest
import torch

from hattention.norm_apis import layer_norm
from hattention.quant_cache_apis import (QuantCache, quant_cache_append, quant_cache_attention,
                                         quant_cache_read, quant_cache_step)
from hattention.rotary_apis import rotary_embedding, rotary_frequencies
from hattention.sliding_apis import sliding_window_attention

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FS = torch.bfloat16, torch.float32
B, H, G, D = 2, 8, 2, 64
N = H * D


def make(seed, *shape, dtype=BF, scale=1.0, shift=0.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=gen) * scale + shift).to(dtype).to(DEV)


def parameters():
    return {"w": make(11, N, dtype=FS, scale=0.1, shift=1.0), "b": make(12, N, dtype=FS, scale=0.1),
            "qkv": make(13, N, (H + 2 * G) * D, scale=N ** -0.5), "out": make(14, N, N, scale=N ** -0.5)}


@functools.lru_cache  # a program makes them once
def FREQS():
    return rotary_frequencies(D // 2, scaling="yarn", factor=4.0, original_length=64, device=DEV)


def project(x, p, positions):
    y = layer_norm(x, p["w"], p["b"])
    q, k, v = (t.unflatten(-1, (-1, D)) for t in (y @ p["qkv"]).split([H * D, G * D, G * D], -1))
    freqs, scale = FREQS()
    q, k = rotary_embedding(q, k, freqs, positions, "half", scale)
    return q, k, v


def train(x, p):
    """The layer as it is trained: every key seen, by a window as long as the sequence."""
    q, k, v = project(x, p, None)
    return x + sliding_window_attention(q, k, v, x.shape[1]).flatten(-2) @ p["out"]


def prompt(x, p, cache, lengths=None):
    """The layer on tokens after those in the cache."""
    q, k, v = project(x, p, cache.counts)
    quant_cache_append(cache, k, v, lengths)
    return x + quant_cache_attention(cache, q, lengths=lengths).flatten(-2) @ p["out"]


def token(x, p, cache):
    q, k, v = project(x, p, cache.counts)
    o, _ = quant_cache_step(cache, q, k, v)
    return x + o.flatten(-2) @ p["out"]


def oracle(x, p):
    """The same layer in 64 bits, by elementary operations, without a cache."""
    c = x - x.mean(-1, keepdim=True)
    y = c / (c.square().mean(-1, keepdim=True) + 1e-5).sqrt() * p["w"] + p["b"]
    q, k, v = (t.unflatten(-1, (-1, D)) for t in (y @ p["qkv"]).split([H * D, G * D, G * D], -1))
    freqs, scale = FREQS()
    n, T = D // 4, x.shape[1]
    angle = (torch.arange(T, device=DEV).double()[:, None] * freqs)[:, None]
    cos, sin = torch.cos(angle) * scale, torch.sin(angle) * scale

    def turn(t):
        a, b = t[..., :n], t[..., n:2 * n]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, t[..., 2 * n:]], -1)
    q, k = turn(q), turn(k)
    q, k, v = (t.transpose(1, 2) for t in (q, k, v))
    k, v = (t.repeat_interleave(H // G, 1) for t in (k, v))
    i = torch.arange(T, device=DEV)
    s = (q @ k.transpose(-1, -2).contiguous() * D ** -0.5).masked_fill(i > i[:, None], -torch.inf)
    return x + (torch.softmax(s, -1) @ v).transpose(1, 2).flatten(-2) @ p["out"]


def apart(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


# A pass rounds to bf16 at most 8 times one after the other (y, qkv, q and k, P, o, its product, the
# sum), each by a relative half step 2^-8 of what it passes on; the gradient goes back through as
# many and was computed from them.  The cache rounds k and v once more, by 2^-4 at most: that
# reaches the layer's addition to the residual stream, which is below the stream itself.
FORWARD, BACKWARD, CACHED = 8 * 2.0 ** -8, 16 * 2.0 ** -8, 8 * 2.0 ** -8 + 2 * 2.0 ** -4


@pytest.mark.parametrize("T", [1, 37, 300])
def test_training_together(T):
    x, p = make(1, B, T, N).requires_grad_(), parameters()
    leaves = [x] + [t.requires_grad_() for t in p.values()]
    do = make(2, B, T, N)
    y = train(x, p)
    grads = torch.autograd.grad(y, leaves, do)
    x64 = x.detach().double().requires_grad_()
    p64 = {n: t.detach().double().requires_grad_() for n, t in p.items()}
    want = oracle(x64, p64)
    ref = torch.autograd.grad(want, [x64, *p64.values()], do.double())
    assert apart(y.detach(), want.detach()) < FORWARD
    for n, a, b in zip(["x", *p], grads, ref):
        assert apart(a, b) < BACKWARD, (n, apart(a, b))


def test_serving_together():
    """A padded batch of prompts, a piece more of each, drafts of which some are dropped, tokens:
    each row as one sequence of its own."""
    p, cache = parameters(), QuantCache.empty(B, G, D, 300, device=DEV)
    first, second, drafts, new = [70, 33], [5, 60], 4, 6
    keep = [3, 1]  # drafted tokens that stay
    total = [a + b + c + new for a, b, c in zip(first, second, keep)]
    full = [make(20 + b, 1, n, N) for b, n in enumerate(total)]
    outs = [[] for _ in range(B)]
    at = [0] * B

    def piece(lens, width):
        x = torch.zeros(B, width, N, dtype=BF, device=DEV)
        for b, n in enumerate(lens):
            x[b, :n] = full[b][0, at[b]:at[b] + n]
        return x

    with torch.no_grad():
        for lens in (first, second):
            y = prompt(piece(lens, max(lens)), p, cache, torch.tensor(lens, device=DEV))
            for b, n in enumerate(lens):
                outs[b].append(y[b, :n])
                at[b] += n
        x = piece(keep, drafts)
        for b, n in enumerate(keep):  # the others are guesses
            x[b, n:] = make(30 + b, drafts - n, N, scale=4.0)
        y = prompt(x, p, cache)
        cache.counts.sub_(torch.tensor([drafts - n for n in keep], device=DEV, dtype=torch.int32))
        for b, n in enumerate(keep):
            outs[b].append(y[b, :n])
            at[b] += n
        for _ in range(new):
            y = token(torch.cat([full[b][:, at[b]] for b in range(B)]), p, cache)
            for b in range(B):
                outs[b].append(y[b:b + 1])
                at[b] += 1
    assert cache.counts.tolist() == total == at
    p64 = {n: t.double() for n, t in p.items()}
    for b in range(B):
        assert apart(torch.cat(outs[b]), oracle(full[b].double(), p64)[0]) < CACHED


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
    q, k = make(1, B, 50, H, D).requires_grad_(), make(2, B, 50, G, D).requires_grad_()
    g = [make(3, B, 50, H, D), make(4, B, 50, G, D)]
    freqs, scale = FREQS()
    at = torch.zeros(B, dtype=torch.int64, device=DEV)

    def step(q=q, k=k):
        y = rotary_embedding(q, k, freqs, at, "interleaved", scale)
        return [*(t.detach() for t in y), *torch.autograd.grad(y, [q, k], g)]
    graph, out = capture(step)
    for i in range(4):
        with torch.no_grad():
            q.copy_(make(10 + i, *q.shape))
            k.copy_(make(20 + i, *k.shape))
            at.fill_(1000 * i)
        graph.replay()
        # other leaves: a graph of the captured ones would outlive the capture
        want = step(q.detach().clone().requires_grad_(), k.detach().clone().requires_grad_())
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_captured_decoding():
    """A captured token, replayed over a block's end, and a captured piece of a prompt: each
    replay advances the cache as an eager call does."""
    p = parameters()
    cache, other = (QuantCache.empty(B, G, D, 512, device=DEV) for _ in range(2))
    x, piece = make(1, B, N), make(2, B, 40, N)
    lens = torch.tensor([40, 7], device=DEV)
    with torch.no_grad():
        one, y = capture(lambda: token(x, p, cache))
        many, z = capture(lambda: prompt(piece, p, cache, lens))
        for t in cache._tensors():
            t.view(torch.uint8).zero_()
        for i in range(70):
            if i % 30 == 7:
                piece.copy_(make(300 + i, B, 40, N))
                many.replay()
                assert torch.equal(z, prompt(piece, p, other, lens))
            x.copy_(make(100 + i, B, N, scale=1 + i % 5))
            one.replay()
            assert torch.equal(y, token(x, p, other)), i
            assert torch.equal(cache.counts, other.counts)
    for a, b in zip(quant_cache_read(cache), quant_cache_read(other)):
        assert torch.equal(a, b)


def test_streams():
    """Calls on a stream of their own, after work that fills it, two at once on caches of their own."""
    p = parameters()
    x = make(1, B, 60, N)
    want = QuantCache.empty(B, G, D, 256, device=DEV)
    with torch.no_grad():
        ref = [prompt(x, p, want), token(x[:, 0], p, want)]
        torch.cuda.synchronize()
        runs = []
        for i in range(2):
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                a = make(5, 2048, 2048)
                for _ in range(20):
                    a = a @ a * 1e-3
                cache = QuantCache.empty(B, G, D, 256, device=DEV)
                runs.append((s, cache, [prompt(x, p, cache), token(x[:, 0], p, cache)]))
        for s, cache, got in runs:
            s.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(ref, got))
            assert torch.equal(cache.counts, want.counts)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="one GPU")
def test_another_device():
    p = {n: t.to("cuda:1") for n, t in parameters().items()}
    cache = QuantCache.empty(B, G, D, 128, device="cuda:1")
    q, k = make(1, B, 9, H, D).to("cuda:1"), make(2, B, 9, G, D).to("cuda:1")
    freqs, _ = rotary_frequencies(D, device="cuda:1")
    q, k = rotary_embedding(q, k, freqs)
    quant_cache_append(cache, k, k)
    assert quant_cache_attention(cache, q).device == q.device and p["w"].device == q.device


def test_mixed_devices():
    q = make(1, B, 9, H, D)
    cache = QuantCache.empty(B, G, D, 128, device=DEV)
    with pytest.raises(RuntimeError):
        rotary_embedding(q, None, rotary_frequencies(D, device="cpu")[0])
    with pytest.raises(RuntimeError):
        quant_cache_attention(cache, q.cpu())
    with pytest.raises(RuntimeError):
        quant_cache_append(cache, q[:, :, :G].cpu(), q[:, :, :G].cpu())
    with pytest.raises(RuntimeError):
        quant_cache_append(cache, q[:, :, :G], q[:, :, :G], torch.tensor([1, 2]))
    with pytest.raises(RuntimeError):
        quant_cache_attention(QuantCache.empty(B, G, D, 128, device="cpu"), q)
