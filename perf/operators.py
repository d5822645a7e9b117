"""The mixers and the norm of a hybrid stack, next to the log-linear scans.

A hybrid model alternates the log-linear layers with sliding-window attention and with
an elementwise gated recurrence, and normalises the residual stream before each.  Each
case is one call, or one training step, that such a program makes:

* ``norm``       layer_norm, alone or with the residual's addition in front of it
* ``rec``        gated_linear_recurrence: h_t = exp(g_t) h_{t-1} + x_t per channel
* ``rec_step``   gated_linear_recurrence_step: one token of it
* ``attn``       sliding_window_attention: a window of keys and a few first tokens
* ``attn_fill``  sliding_window_prefill: the same over a padded batch of prompts, ready to decode
* ``attn_step``  sliding_window_step: one token against the window's cache

With ``own`` false ``run`` computes a case in elementary torch operations, with ``own``
true through the package.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5


# --------------------------------------------------------------------------
# the cases
# --------------------------------------------------------------------------
def listed():
    return [
        # the norm before a layer while decoding 64 users: latency
        dict(name="norm_decode", kind="norm", rows=64, n=1024, dtype="bf16", params="bf16",
             residual=True, train=False),
        # the norm of a training step, 4 x 16384 tokens, with the residual stream's sum
        dict(name="norm_train", kind="norm", rows=65536, n=1024, dtype="bf16", params="fp32",
             residual=True, train=True),
        # a wider one in full precision, a number of rows that no tile divides
        dict(name="norm_train_fp32", kind="norm", rows=8190, n=2304, dtype="fp32", params="fp32",
             residual=False, train=True),
        # one token of the recurrence for 64 users: latency
        dict(name="rec_step", kind="rec_step", B=64, D=2048, dtype="bf16", gates="fp32"),
        # the training step of a recurrent layer
        dict(name="rec_train", kind="rec", B=4, T=8192, D=2048, dtype="bf16", gates="bf16",
             train=True, state=False, ragged=False),
        # evaluation of one long document in full precision: few channels, a long axis
        dict(name="rec_long", kind="rec", B=1, T=131072, D=1024, dtype="fp32", gates="fp32",
             train=False, state=False, ragged=False),
        # a padded batch that goes on from a state and is trained through it
        dict(name="rec_train_state", kind="rec", B=3, T=4005, D=1000, dtype="fp16", gates="fp32",
             train=True, state=True, ragged=True),
        # one token for one user against a window of 1024: latency
        dict(name="attn_step_one", kind="attn_step", B=1, H=16, G=4, D=64, window=1024, sinks=4,
             seen=700, dtype="bf16"),
        # one token for 64 users, some of them still inside their first window
        dict(name="attn_step", kind="attn_step", B=64, H=32, G=8, D=128, window=4096, sinks=4,
             seen=9000, dtype="bf16"),
        # prompts of several lengths whose last window decoding goes on from
        dict(name="attn_fill", kind="attn_fill", B=4, T=4005, H=16, G=2, D=128, window=512,
             sinks=4, dtype="fp16", ragged=True),
        # the training step of an attention layer between scan layers, heads of 64
        dict(name="attn_train", kind="attn", B=4, T=8192, H=16, G=16, D=64, window=1024, sinks=4,
             dtype="bf16", train=True, ragged=False),
        # heads of 128 in groups, one long sequence, a wide window
        dict(name="attn_train_wide", kind="attn", B=1, T=16384, H=16, G=4, D=128, window=4096,
             sinks=16, dtype="bf16", train=True, ragged=False),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_COST = {  # the most that a drawn case of each kind may take: bytes, operations
    "norm": (1.3e9, 1e11), "rec": (1.7e9, 1e11), "rec_step": (4e6, 1e9),
    "attn_step": (7e8, 1e11), "attn_fill": (3e8, 2e11), "attn": (4e8, 1.9e12)}


def draw(rng):
    kind = rng.choice(["norm", "norm", "rec", "rec", "rec_step", "attn", "attn", "attn",
                       "attn_fill", "attn_step", "attn_step"])
    wide, half = ["bf16", "bf16", "fp16", "fp32"], ["bf16", "bf16", "fp16"]
    while True:
        dtype = rng.choice(wide if kind in ("norm", "rec", "rec_step") else half)
        c = dict(kind=kind)
        if kind == "norm":
            n = rng.choice([_log(rng, 16, 8192), 8 * _log(rng, 2, 1024), 64 * _log(rng, 1, 64)])
            c.update(rows=_log(rng, 1, 65536), n=n, dtype=dtype,
                     params=rng.choice(["fp32", dtype]), residual=rng.random() < 0.6,
                     train=rng.random() < 0.7)
        elif kind == "rec":
            c.update(B=_log(rng, 1, 8), T=_log(rng, 1, 131072),
                     D=rng.choice([_log(rng, 1, 4096), 64 * _log(rng, 1, 64)]), dtype=dtype,
                     gates=rng.choice(["fp32", dtype]), train=rng.random() < 0.6,
                     state=rng.random() < 0.4, ragged=rng.random() < 0.3)
        elif kind == "rec_step":
            c.update(B=_log(rng, 1, 256), D=_log(rng, 64, 4096), dtype=dtype,
                     gates=rng.choice(["fp32", dtype]))
        else:
            G = _log(rng, 1, 16)
            c.update(B=_log(rng, 1, 64 if kind == "attn_step" else 8), G=G,
                     H=G * rng.choice([1, 1, 2, 4, 8]), D=rng.choice([64, 128, 64, 128, 80, 96]),
                     window=_log(rng, 1, 4096), sinks=rng.choice([0, 1, 4, 16, 64]), dtype=dtype)
            if kind == "attn_step":
                c.update(seen=_log(rng, 1, 16384))
            else:
                c.update(T=_log(rng, 1, 16384), ragged=rng.random() < 0.4)
            if kind == "attn":
                c.update(train=rng.random() < 0.7)
        w = work(c)
        if w["bytes"] <= _COST[kind][0] and w["flops"] <= _COST[kind][1]:
            return c


def _lengths(c):
    """Tokens of each row of a padded batch: the first is full, the last about half."""
    B, T = c["B"], c["T"]
    return [T - b * T // (2 * B) for b in range(B)]


def _seen(c):
    """Tokens that each row of a decoding batch has seen."""
    return [1 + (b + 1) * (c["seen"] - 1) // c["B"] for b in range(c["B"])]


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
class _Make:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(DEV).manual_seed(seed)

    def normal(self, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
        x = torch.randn(*shape, generator=self.gen, device=DEV)
        return x.mul_(scale).add_(shift).to(dtype)

    def decay(self, *shape, dtype):
        """Log-decays: channels that remember from one token to about a thousand,
        each token's gate about its channel's."""
        rate = torch.rand(shape[-1], generator=self.gen, device=DEV).mul_(math.log(1e3)).neg_().exp_()
        x = torch.randn(*shape, generator=self.gen, device=DEV).mul_(0.5).exp_()
        return x.mul_(rate).neg_().to(dtype)


def prepare(case, seed):
    c, m, dt = case, _Make(seed), DTYPES[case["dtype"]]
    kind = c["kind"]
    s, x = dict(case=dict(c)), {}
    if kind == "norm":
        rows, n, pdt = c["rows"], c["n"], DTYPES[c["params"]]
        x["x"] = m.normal(rows, n, dtype=dt)
        x["weight"] = m.normal(n, dtype=pdt, scale=0.1, shift=1.0)
        x["bias"] = m.normal(n, dtype=pdt, scale=0.1)
        if c["residual"]:
            x["residual"] = m.normal(rows, n, dtype=dt, scale=3.0, shift=0.2)
        if c["train"]:
            s["dy"] = m.normal(rows, n, dtype=dt)
            s["ds"] = m.normal(rows, n, dtype=dt) if c["residual"] else None
    elif kind == "rec":
        B, T, D = c["B"], c["T"], c["D"]
        x["x"] = m.normal(B, T, D, dtype=dt)
        x["g"] = m.decay(B, T, D, dtype=DTYPES[c["gates"]])
        if c["state"]:
            x["initial_state"] = m.normal(B, D, scale=2.0)
        if c["train"]:
            s["do"] = m.normal(B, T, D, dtype=dt)
            s["dht"] = m.normal(B, D) if c["state"] else None
        if c["ragged"]:
            s["lengths"] = torch.tensor(_lengths(c), dtype=torch.int32, device=DEV)
    elif kind == "rec_step":
        x["x"] = m.normal(c["B"], c["D"], dtype=dt)
        x["g"] = m.decay(c["B"], c["D"], dtype=DTYPES[c["gates"]])
        x["state"] = m.normal(c["B"], c["D"], scale=3.0)
    elif kind == "attn_step":
        B, H, G, D = c["B"], c["H"], c["G"], c["D"]
        slots = c["sinks"] + c["window"]
        x["q"] = m.normal(B, H, D, dtype=dt)
        x["k"] = m.normal(B, G, D, dtype=dt)
        x["v"] = m.normal(B, G, D, dtype=dt)
        x["k_cache"] = m.normal(B, G, slots, D, dtype=dt)
        x["v_cache"] = m.normal(B, G, slots, D, dtype=dt)
        x["counts"] = torch.tensor(_seen(c), dtype=torch.int32, device=DEV)
    else:
        B, T, H, G, D = c["B"], c["T"], c["H"], c["G"], c["D"]
        x["q"] = m.normal(B, T, H, D, dtype=dt)
        x["k"] = m.normal(B, T, G, D, dtype=dt)
        x["v"] = m.normal(B, T, G, D, dtype=dt)
        if c.get("train"):
            s["do"] = m.normal(B, T, H, D, dtype=dt)
        if c["ragged"]:
            s["lengths"] = torch.tensor(_lengths(c), dtype=torch.int32, device=DEV)
    if c.get("train"):
        for t in x.values():
            t.requires_grad_()
    s["x"] = x
    return s


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def _ours():
    """The package's entry points."""
    root = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..")
    sys.path.insert(0, os.path.join(root, "log-linear-attention_amd"))
    from hattention import norm_apis, recurrence_apis, sliding_apis
    return norm_apis, recurrence_apis, sliding_apis


_apis = None


def run(state):
    global _apis
    c, x = state["case"], state["x"]
    kind = c["kind"]
    if own:
        if _apis is None:
            _apis = _ours()
        norm, rec, att = _apis
    if kind == "rec_step":
        if own:
            o, h = rec.gated_linear_recurrence_step(x["state"], x["x"], x["g"])
        else:
            o, h = _plain_rec_step(**x)
        return {"o": o, "state": h}
    if kind == "attn_step":
        if own:
            S = att.SlidingState(x["k_cache"], x["v_cache"], x["counts"], c["window"], c["sinks"])
            o, S = att.sliding_window_step(S, x["q"], x["k"], x["v"])
        else:
            o = _plain_attn_step(**x, window=c["window"], sinks=c["sinks"])
        return {"o": o, "k": x["k_cache"], "v": x["v_cache"], "counts": x["counts"]}
    if kind == "attn_fill":
        if own:
            o, S = att.sliding_window_prefill(x["q"], x["k"], x["v"], c["window"], c["sinks"],
                                              lengths=state.get("lengths"))
            return {"o": o, "k": S.k, "v": S.v, "counts": S.counts}
        return _plain_attn_fill(x, c, state.get("lengths"))
    with torch.set_grad_enabled(bool(c["train"])):
        if kind == "norm":
            f = norm.layer_norm if own else _plain_norm
            out = f(x["x"], x["weight"], x["bias"], residual=x.get("residual"), eps=EPS)
            outs = dict(zip("ys", out)) if c["residual"] else {"y": out}
        elif kind == "rec":
            f = rec.gated_linear_recurrence if own else _plain_rec
            out = f(x["x"], x["g"], initial_state=x.get("initial_state"),
                    output_final_state=c["state"], lengths=state.get("lengths"))
            outs = dict(o=out[0], ht=out[1]) if c["state"] else {"o": out}
        else:
            f = att.sliding_window_attention if own else _plain_attn
            outs = {"o": f(x["q"], x["k"], x["v"], c["window"], c["sinks"],
                           lengths=state.get("lengths"))}
    if not c["train"]:
        return outs
    grads = torch.autograd.grad(list(outs.values()), list(x.values()),
                                [state["d" + n] for n in outs])
    return {**outs, **{"d" + n: t for n, t in zip(x, grads)}}


# --------------------------------------------------------------------------
# the plain forms
# --------------------------------------------------------------------------
def _plain_norm(x, weight, bias, residual, eps):
    y, s = _PlainNorm.apply(x, weight, bias, residual, eps)
    return (y, s) if residual is not None else y


class _PlainNorm(torch.autograd.Function):
    """y = (s - mean) rstd weight + bias in 32 bits, the parameters' sums in 64. s = x +
    residual is what the residual stream holds, so the norm is of the rounded sum."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps):
        s = x if residual is None else (x.float() + residual.float()).to(residual.dtype)
        f = s.float()
        f = f - f.mean(-1, keepdim=True)
        rstd = torch.rsqrt(f.square().mean(-1, keepdim=True) + eps)
        hat = f * rstd
        ctx.save_for_backward(hat, rstd, weight)
        ctx.types = x.dtype, bias.dtype, None if residual is None else residual.dtype
        return (hat * weight.float() + bias.float()).to(x.dtype), s if residual is not None else None

    @staticmethod
    def backward(ctx, dy, ds):
        hat, rstd, weight = ctx.saved_tensors
        xt, bt, rt = ctx.types
        dy = dy.float()
        dw = (dy * hat).sum(0, dtype=torch.float64)
        db = dy.sum(0, dtype=torch.float64)
        t = dy * weight.float()
        dx = rstd * (t - t.mean(-1, keepdim=True) - hat * (t * hat).mean(-1, keepdim=True))
        if rt is not None:
            dx = dx + ds.float()
        return (dx.to(xt), dw.to(weight.dtype), db.to(bt), dx.to(rt) if rt is not None else None,
                None)


def _doubling(a, b):
    """h_t = a_t h_{t-1} + b_t over axis 1 (h_{-1} = 0), by doubling: after the step of
    width w, (a, b) of a token stand for the last 2 w tokens up to it."""
    w = 1
    while w < b.shape[1]:
        b = torch.cat([b[:, :w], b[:, w:] + a[:, w:] * b[:, :-w]], 1)
        a = torch.cat([a[:, :w], a[:, w:] * a[:, :-w]], 1)
        w *= 2
    return b


def _live(lengths, B, T):
    """[B, T]: the tokens that are not padding."""
    t = torch.arange(T, device=DEV)
    return (t < lengths[:, None]) if lengths is not None else (t >= 0).expand(B, T)


def _plain_rec(x, g, initial_state, output_final_state, lengths):
    o, ht = _PlainRec.apply(x, g, initial_state, lengths)
    return (o, ht) if output_final_state else o


class _PlainRec(torch.autograd.Function):
    """Padding has a = 1 and adds nothing, so the state of the last token is the final one."""

    @staticmethod
    def forward(ctx, x, g, h0, lengths):
        B, T, D = x.shape
        live = _live(lengths, B, T)[..., None]
        a = torch.where(live, g.float().exp(), 1.0)
        b = torch.where(live, x.float(), 0.0)
        if h0 is not None:
            b = torch.cat([b[:, :1] + a[:, :1] * h0[:, None], b[:, 1:]], 1)
        h = _doubling(a, b)
        ctx.save_for_backward(a, h, h0, live)
        ctx.types = x.dtype, g.dtype
        return torch.where(live, h, 0.0).to(x.dtype), h[:, -1].clone()

    @staticmethod
    def backward(ctx, do, dht):
        a, h, h0, live = ctx.saved_tensors
        xt, gt = ctx.types
        d = torch.where(live, do.float(), 0.0)
        if dht is not None:
            d = torch.cat([d[:, :-1], d[:, -1:] + dht[:, None]], 1)
        after = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1)
        dh = _doubling(after.flip(1), d.flip(1)).flip(1)
        first = (h0 if h0 is not None else torch.zeros_like(h[:, 0]))[:, None]
        dg = dh * a * torch.cat([first, h[:, :-1]], 1)
        return (torch.where(live, dh, 0.0).to(xt), torch.where(live, dg, 0.0).to(gt),
                dh[:, 0] * a[:, 0] if h0 is not None else None, None)


def _plain_rec_step(x, g, state):
    state.copy_(g.float().exp() * state + x.float())
    return state.to(x.dtype), state


def _plain_attn(q, k, v, window, sinks, lengths=None):
    """Blocks of C queries against the C + window keys that any of them sees, and the
    first tokens beside them where they lie before the window."""
    B, T, H, D = q.shape
    G, R = k.shape[2], H // k.shape[2]
    C = max(16, min(512, T))
    n = -(-T // C)
    W = min(window, T)
    band = C + W
    pad = torch.nn.functional.pad
    heads = lambda t: t.float().transpose(1, 2)                           # [B, heads, T, D]
    qb = pad(heads(q), (0, 0, 0, n * C - T)).reshape(B, G, R, n, C, D)
    qb = qb.transpose(2, 3).reshape(B, G, n, R * C, D) * D ** -0.5
    # block i has the keys from i C - W to i C + C - 1
    kh, vh = heads(k), heads(v)
    kb, vb = (pad(t, (0, 0, W, n * C - T)).unfold(2, band, C).transpose(-1, -2)
              for t in (kh, vh))                                          # [B, G, n, band, D]
    first = min(sinks, T)
    kf, vf = (t[:, :, None, :first].expand(B, G, n, first, D) for t in (kh, vh))
    t = torch.arange(n * C, device=DEV).view(n, C, 1)
    s = torch.arange(n, device=DEV).view(n, 1, 1) * C - W + torch.arange(band, device=DEV)
    f = torch.arange(first, device=DEV)
    end = lengths if lengths is not None else torch.full((B,), T, device=DEV)
    end = end.view(B, 1, 1, 1)
    seen = torch.cat([((s >= 0) & (s <= t) & (s > t - W))[None] & (s < end) & (t < end),
                      ((f <= t) & (f <= t - W))[None] & (f < end) & (t < end)], -1)
    seen = seen[:, None, :, None].expand(B, 1, n, R, C, band + first).reshape(
        B, 1, n, R * C, band + first)
    p = torch.cat([qb @ kb.transpose(-1, -2), qb @ kf.transpose(-1, -2)], -1)
    p = torch.where(seen, p, -1e30)
    p = torch.where(seen, (p - p.amax(-1, keepdim=True).detach()).exp(), 0.0)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    o = p[..., :band] @ vb + p[..., band:] @ vf
    o = o.view(B, G, n, R, C, D).transpose(2, 3).reshape(B, H, n * C, D)[:, :, :T]
    return o.transpose(1, 2).to(q.dtype)


def _plain_attn_fill(x, c, lengths):
    q, k, v, W, S = x["q"], x["k"], x["v"], c["window"], c["sinks"]
    B, T = q.shape[:2]
    end = lengths if lengths is not None else torch.full((B,), T, dtype=torch.int32, device=DEV)
    # slot S + i of the window holds the last token whose position is S + i modulo W
    i = torch.arange(S + W, device=DEV)
    last = end.long()[:, None] - 1
    at = torch.where(i < S, i, last - (last - i) % W)
    held = (at <= last) & (at >= torch.where(i < S, 0, S))
    rows = torch.arange(B, device=DEV)[:, None]

    def cache(t):
        t = t[rows, at.clamp(0, T - 1)]                                   # [B, slots, G, D]
        return torch.where(held[..., None, None], t, 0).transpose(1, 2).contiguous()
    return {"o": _plain_attn(q, k, v, W, S, lengths), "k": cache(k), "v": cache(v),
            "counts": end.clone()}


def _plain_attn_step(q, k, v, k_cache, v_cache, counts, window, sinks):
    B, H, D = q.shape
    G, slots = k_cache.shape[1], k_cache.shape[2]
    n = counts.long()
    at = torch.where(n < sinks, n, sinks + (n - sinks) % window)
    rows = torch.arange(B, device=DEV)
    k_cache[rows, :, at] = k
    v_cache[rows, :, at] = v
    counts += 1
    held = torch.arange(slots, device=DEV) < counts[:, None]
    p = (q.float() * D ** -0.5).view(B, G, H // G, D) @ k_cache.float().transpose(-1, -2)
    p = torch.where(held[:, None, None], p, -1e30)
    p = (p - p.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    return (p @ v_cache.float()).view(B, H, D).to(q.dtype)


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def _pairs(T, W, S):
    """Keys seen by the T queries of one row: min(t + 1, W), and the first tokens that
    lie before the window."""
    full = max(0, T - W)
    near = min(T, W) * (min(T, W) + 1) // 2 + full * W
    m = min(S, full)
    return near + m * (m + 1) // 2 + (full - m) * S


def work(case):
    c = case
    kind, e = c["kind"], DTYPES[c["dtype"]].itemsize
    if kind == "norm":
        p = DTYPES[c["params"]].itemsize
        streams = 2 + (2 if c["residual"] else 0)
        if c["train"]:
            streams += 2 + (2 if c["residual"] else 0)       # dy, dx; ds, dresidual
        return dict(bytes=c["rows"] * c["n"] * e * streams + c["n"] * p * (4 if c["train"] else 2),
                    flops=c["rows"] * c["n"] * (24 if c["train"] else 8))
    if kind in ("rec", "rec_step"):
        ge = DTYPES[c["gates"]].itemsize
        if kind == "rec_step":
            return dict(bytes=c["B"] * c["D"] * (2 * e + ge + 8), flops=3 * c["B"] * c["D"])
        tokens = sum(_lengths(c)) if c["ragged"] else c["B"] * c["T"]
        full = c["B"] * c["T"]
        ins, outs = e + ge, e
        if c["train"]:
            ins, outs = ins + e, outs + e + ge
        ends = (2 * (2 if c["train"] else 1)) * c["B"] * c["D"] * 4 if c["state"] else 0
        return dict(bytes=c["D"] * (tokens * ins + full * outs) + ends,
                    flops=c["D"] * tokens * (9 if c["train"] else 3))
    B, H, G, D, W, S = (c[n] for n in ("B", "H", "G", "D", "window", "sinks"))
    if kind == "attn_step":
        keys = sum(min(n + 1, S + W) for n in _seen(c))
        return dict(bytes=2 * keys * G * D * e + B * (2 * H + 2 * G) * D * e, flops=4 * keys * H * D)
    T = c["T"]
    lens = _lengths(c) if c["ragged"] else [T] * B
    pairs = sum(_pairs(n, W, S) for n in lens)
    tokens = sum(lens)
    nbytes = tokens * (H + 2 * G) * D * e + B * T * H * D * e
    flops = 4 * D * H * pairs
    if kind == "attn_fill":
        nbytes += 2 * B * G * (S + W) * D * e
    elif c["train"]:
        nbytes += tokens * H * D * e + B * T * (H + 2 * G) * D * e
        flops += 10 * D * H * pairs
    return dict(bytes=nbytes, flops=flops)


# --------------------------------------------------------------------------
# the same results from the definitions, in 64 bits
# --------------------------------------------------------------------------
def exact(case, seed):
    c = case
    s = prepare(c, seed)
    x = {n: t.detach() for n, t in s["x"].items()}
    with torch.no_grad():
        if c["kind"] == "norm":
            return _exact_norm(c, s, x)
        if c["kind"] == "rec":
            return _exact_rec(c, s, x)
        if c["kind"] == "rec_step":
            h = torch.exp(x["g"].double()) * x["state"].double() + x["x"].double()
            return {"o": h, "state": h}
        if c["kind"] == "attn_step":
            return _exact_attn_step(c, x)
        return _exact_attn(c, s, x)


def _exact_norm(c, s, x):
    base = x["x"].double()
    if c["residual"]:
        base = (base + x["residual"].double()).to(x["residual"].dtype).double()
    n = c["n"]
    mean = base.sum(1) / n
    var = ((base - mean[:, None]) ** 2).sum(1) / n
    hat = (base - mean[:, None]) / torch.sqrt(var + EPS)[:, None]
    w = x["weight"].double()
    out = {"y": w * hat + x["bias"].double()}
    if c["residual"]:
        out["s"] = base
    if c["train"]:
        dy = s["dy"].double()
        dhat = dy * w
        # the norm's derivative: what is left of dhat across the ones and hat
        dx = dhat - dhat.sum(1)[:, None] / n - hat * ((dhat * hat).sum(1) / n)[:, None]
        dx = dx / torch.sqrt(var + EPS)[:, None]
        if c["residual"]:
            dx = dx + s["ds"].double()
            out["dresidual"] = dx
        out.update(dx=dx, dweight=(dy * hat).sum(0), dbias=dy.sum(0))
    return out


def _exact_rec(c, s, x):
    B, T, D = c["B"], c["T"], c["D"]
    if B * T * D > 2 ** 28:
        return None
    lens = _lengths(c) if c["ragged"] else [T] * B
    a = torch.exp(x["g"].double())
    b = x["x"].double()
    h = torch.zeros(B, T + 1, D, dtype=torch.float64, device=DEV)
    if c["state"]:
        h[:, 0] = x["initial_state"]
    for t in range(T):
        torch.addcmul(b[:, t], a[:, t], h[:, t], out=h[:, t + 1])
    out = {"o": h[:, 1:].clone()}
    for i, n in enumerate(lens):
        out["o"][i, n:] = 0
    if c["state"]:
        out["ht"] = torch.stack([h[i, n] for i, n in enumerate(lens)])
    if c["train"]:
        do = s["do"].double()
        live = torch.arange(T, device=DEV)[:, None] < torch.tensor(lens, device=DEV)[:, None, None]
        dh = do.masked_fill(~live, 0.0)
        d = s["dht"].double() if c["state"] else torch.zeros_like(h[:, 0])
        for t in range(T - 1, -1, -1):
            torch.add(d, dh[:, t], out=dh[:, t])
            d = torch.where(live[:, t], dh[:, t] * a[:, t], d)
        out["dx"] = dh.masked_fill(~live, 0.0)
        out["dg"] = out["dx"] * a * h[:, :-1]
        if c["state"]:
            out["dinitial_state"] = d
    return out


def _exact_attn(c, s, x):
    B, T, H, G, D, W, S = (c[n] for n in ("B", "T", "H", "G", "D", "window", "sinks"))
    R, train = H // G, c.get("train", False)
    lens = _lengths(c) if c["ragged"] else [T] * B
    zeros = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=DEV)
    o = zeros(x["q"])
    dq, dk, dv = (zeros(x[n]) for n in "qkv")
    i = torch.arange(T, device=DEV)
    ahead = i[:, None] - i
    hidden = (ahead < 0) | ((ahead >= W) & (i >= S))
    for b, n in enumerate(lens):
        for h in range(H):
            q, k, v = (x[m][b, :n, j].double() for m, j in (("q", h), ("k", h // R), ("v", h // R)))
            p = torch.softmax((q @ k.T / math.sqrt(D)).masked_fill_(hidden[:n, :n], -math.inf), 1)
            o[b, :n, h] = p @ v
            if train:
                do = s["do"][b, :n, h].double()
                dv[b, :n, h // R] += p.T @ do
                dp = do @ v.T
                ds = p * dp.sub_((p * dp).sum(1, keepdim=True)) / math.sqrt(D)
                dq[b, :n, h] = ds @ k
                dk[b, :n, h // R] += ds.T @ q
    out = {"o": o}
    if train:
        out.update(dq=dq, dk=dk, dv=dv)
    if c["kind"] == "attn_fill":
        for m in "kv":
            out[m] = torch.zeros(B, G, S + W, D, dtype=torch.float64, device=DEV)
            for b, n in enumerate(lens):
                out[m][b, :, :min(S, n)] = x[m][b, :min(S, n)].double().transpose(0, 1)
                for t in range(max(S, n - W), n):
                    out[m][b, :, S + (t - S) % W] = x[m][b, t].double()
        out["counts"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    return out


def _exact_attn_step(c, x):
    W, S, D = c["window"], c["sinks"], c["D"]
    kc, vc = x["k_cache"].double(), x["v_cache"].double()
    o = torch.zeros(c["B"], c["H"], D, dtype=torch.float64, device=DEV)
    for b, n in enumerate(_seen(c)):
        slot = n if n < S else S + (n - S) % W
        kc[b, :, slot], vc[b, :, slot] = x["k"][b].double(), x["v"][b].double()
        m = min(n + 1, S + W)
        for h in range(c["H"]):
            g = h // (c["H"] // c["G"])
            p = torch.softmax(kc[b, g, :m] @ x["q"][b, h].double() / math.sqrt(D), 0)
            o[b, h] = p @ vc[b, g, :m]
    return {"o": o, "k": kc, "v": vc, "counts": x["counts"] + 1}
