"""gated_linear_recurrence where a state or a gradient is not finite: h_t = exp(g_t) h_{t-1} + x_t
keeps it, however far the product of the decays underflows (0 < exp(g): inf stays inf, NaN stays
NaN; exp(-inf) = 0, and 0 times either is NaN)."""
import pytest
import torch

from hattention.recurrence_apis import gated_linear_recurrence

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
INF, NAN = float("inf"), float("nan")
# the product over a segment (128 or 256 tokens) of exp(-1) is below the smallest fp32 number
B, T, D, AT = 2, 1300, 70, 11


def make(seed, *shape, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=gen).to(dtype).to(DEV)


def decays(dtype):
    g = torch.full((B, T, D), -1.0, device=DEV, dtype=dtype)
    g[..., 1::2] = -1e-3  # slow channels beside the fast ones
    return g


DTYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
          (torch.float16, torch.float32)]


@pytest.mark.parametrize("xt,gt", DTYPES)
@pytest.mark.parametrize("what", [INF, -INF, NAN])
def test_a_state_that_is_not_finite_stays(xt, gt, what):
    x, g, h0 = make(1, B, T, D, dtype=xt), decays(gt), make(2, B, D)
    base, hbase = gated_linear_recurrence(x, g, h0, True)
    x2, h2 = x.clone(), h0.clone()
    x2[1, AT, 4], x2[1, AT, 5] = what, what
    h2[0, 8], h2[0, 9] = what, what
    o, ht = gated_linear_recurrence(x2, g, h2, True)
    is_what = (lambda t: t.isnan()) if what != what else (lambda t: t == what)
    for b, d, start in ((1, 4, AT), (1, 5, AT), (0, 8, 0), (0, 9, 0)):
        assert is_what(o[b, start:, d]).all(), (b, d, int((~is_what(o[b, start:, d])).nonzero()[0]))
        assert is_what(ht[b, d])
        assert torch.equal(o[b, :start, d], base[b, :start, d])
        o[b, :, d], ht[b, d] = base[b, :, d], hbase[b, d]
    assert torch.equal(o, base) and torch.equal(ht, hbase)


@pytest.mark.parametrize("xt,gt", DTYPES)
@pytest.mark.parametrize("what", [INF, NAN])
def test_a_gradient_that_is_not_finite_stays(xt, gt, what):
    x, g, h0 = (t.requires_grad_() for t in (make(1, B, T, D, dtype=xt), decays(gt), make(2, B, D)))
    do, dht = make(3, B, T, D, dtype=xt), make(4, B, D)
    grads = lambda do, dht: torch.autograd.grad(gated_linear_recurrence(x, g, h0, True),
                                                [x, g, h0], [do, dht])
    base = grads(do, dht)
    do2, dht2 = do.clone(), dht.clone()
    end = T - AT
    do2[1, end, 4], do2[1, end, 5] = what, what
    dht2[0, 8], dht2[0, 9] = what, what
    got = grads(do2, dht2)
    is_what = (lambda t: t.isnan()) if what != what else (lambda t: t == what)
    for b, d, n in ((1, 4, end + 1), (1, 5, end + 1), (0, 8, T), (0, 9, T)):
        assert is_what(got[0][b, :n, d]).all(), (b, d, int((~is_what(got[0][b, :n, d])).sum()))
        assert not got[1][b, :n, d].isfinite().any()  # times a state of either sign
        assert is_what(got[2][b, d])
        for a, z in zip(got[:2], base[:2]):
            assert torch.equal(a[b, n:, d], z[b, n:, d])
            a[b, :, d] = z[b, :, d]
        got[2][b, d] = base[2][b, d]
    assert all(torch.equal(a, z) for a, z in zip(got, base))


@pytest.mark.parametrize("xt,gt", DTYPES)
def test_a_reset_keeps_nan(xt, gt):
    """exp(-inf) = 0 forgets a finite state to the bit; 0 times NaN or infinity is NaN, in the
    token loop as across segments."""
    x, g = make(1, B, T, D, dtype=xt), decays(gt)
    g[:, [300, 777]] = -INF
    o, ht = gated_linear_recurrence(x, g, None, True)
    assert torch.equal(o[:, 777], x[:, 777]) and o.isfinite().all()
    x[0, AT, 4], x[0, AT, 5] = NAN, INF
    o2, ht2 = gated_linear_recurrence(x, g, None, True)
    assert o2[0, AT:, 4].isnan().all() and ht2[0, 4].isnan()
    assert (o2[0, AT:300, 5] == INF).all() and o2[0, 300:, 5].isnan().all() and ht2[0, 5].isnan()
    keep = [d for d in range(D) if d not in (4, 5)]
    assert torch.equal(o[..., keep], o2[..., keep]) and torch.equal(o[1], o2[1])
