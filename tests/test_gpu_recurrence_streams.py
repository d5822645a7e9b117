"""Recurrences larger than the card (more workgroups than it holds at once) that run at the same
time on two streams: neither's segments may wait for workgroups that the other keeps from
starting.  The bits do not depend on timing, so they are those of a call alone."""
import pytest
import torch

from hattention.recurrence_apis import gated_linear_recurrence

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
B, T, D = 4, 8192, 2048  # 4096 workgroups of 512 threads; at most two of them fit a CU


def make(seed, dtype):
    gen = torch.Generator(DEV).manual_seed(seed)
    draw = lambda: torch.randn(B, T, D, generator=gen, device=DEV)
    rate = torch.exp(-7 * torch.rand(D, generator=gen, device=DEV))
    x, g, do = draw().to(dtype), (-rate * torch.exp(0.5 * draw())).to(dtype), draw().to(dtype)
    return x.requires_grad_(), g.requires_grad_(), do


def step(x, g, do):
    o, ht = gated_linear_recurrence(x, g, None, True)
    return [o.detach(), ht.detach(), *torch.autograd.grad(o, [x, g], do)]


def test_two_streams_each_larger_than_the_card():
    ins = [make(1, torch.bfloat16), make(2, torch.bfloat16)]
    want = [step(*t) for t in ins]
    assert all(z.isfinite().all() for w in want for z in w)
    streams = [torch.cuda.Stream() for _ in ins]
    torch.cuda.synchronize()
    for turn in range(3):
        got = []
        for t, s in zip(ins, streams):
            with torch.cuda.stream(s):
                got.append(step(*t))
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(got, want)):
            for name, u, v in zip(("o", "ht", "dx", "dg"), a, b):
                assert torch.equal(u, v), (turn, i, name)


def test_replays_take_every_segment():
    """The counter that hands out the segments starts again with each replay."""
    x, g = (t[:1, :2000, :200].detach().contiguous() for t in make(3, torch.bfloat16)[:2])
    other = make(4, torch.bfloat16)[0][:1, :2000, :200].detach().contiguous()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gated_linear_recurrence(x, g, None, True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, ht = gated_linear_recurrence(x, g, None, True)
    for turn in range(4):
        x.copy_(other * (turn + 1))
        want = gated_linear_recurrence(x, g, None, True)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want[0]) and torch.equal(ht, want[1]), turn
