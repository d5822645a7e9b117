"""Global attention beside the log-linear scans: rotary positions, a cache held in 8 bits,
and the attention over it.

The few global attention layers of a hybrid stack rotate q and k by their positions, keep k
and v of all tokens (codes of 8 bits, a scale for each 64 tokens of a head), and attend over
that cache: a chunk of a prompt, a few drafted tokens, or one token a row.  Each case is one
call, or one training step, that such a program makes:

* ``rope``    rotary_embedding of q and k, forward or forward and backward
* ``append``  quant_cache_append: new tokens of each row enter the cache
* ``read``    quant_cache_read: the tokens back in 16 or 32 bits
* ``attn``    quant_cache_attention: the last T tokens of each row against the cache
* ``step``    quant_cache_step: one token a row, entering the cache and attending over it

With ``own`` false ``run`` computes a case in elementary torch operations, with ``own``
true through the package.  A pass that appends first sets the counts back to the tokens that
were there, as a program does that takes rows into use again.
"""
import math
import os
import random
import sys

import torch

own = False
DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn
BLOCK = 64                                  # tokens that share a scale
LEAST = -100                                # the least exponent of a scale
MOST = {"bf16": 119, "fp16": 7}             # the largest: 448 times it stays finite in the type


# --------------------------------------------------------------------------
# the cases
# --------------------------------------------------------------------------
def listed():
    return [
        # q and k of one token of 64 users: latency
        dict(name="rope_decode", kind="rope", B=64, T=1, H=32, G=8, D=128, rot=128, layout="half",
             scale=1.0, positions="row", seen=9000, dtype="bf16", train=False),
        # the training step of a layer, 4 x 8192 tokens
        dict(name="rope_train", kind="rope", B=4, T=8192, H=16, G=16, D=64, rot=64, layout="half",
             scale=1.0, positions="none", seen=0, dtype="bf16", train=True),
        # packed documents in full precision, a quarter of the head rotated, far positions,
        # frequencies of a longer context
        dict(name="rope_train_part", kind="rope", B=1, T=8005, H=12, G=4, D=128, rot=32,
             layout="interleaved", scale=1.2, positions="token", seen=500000, dtype="fp32",
             train=True),
        # prompts of several lengths enter an empty cache
        dict(name="append_prompt", kind="append", B=4, T=8192, G=8, D=128, seen=0, dtype="bf16",
             ragged=True),
        # the next piece of 16 prompts, from the middle of a block on
        dict(name="append_chunk", kind="append", B=16, T=301, G=4, D=96, seen=1000, dtype="fp16",
             ragged=True),
        # the whole cache of 8 users back in 16 bits
        dict(name="read", kind="read", B=8, G=8, D=128, seen=16000, start=0, n=16000, dtype="bf16"),
        # a window of it in 32 bits
        dict(name="read_part", kind="read", B=3, G=2, D=80, seen=5000, start=1003, n=777,
             dtype="fp32"),
        # one token for one user: latency
        dict(name="step_one", kind="step", B=1, H=16, G=4, D=64, seen=700, dtype="bf16"),
        # one token for 64 users, of a few tokens to 9000
        dict(name="step", kind="step", B=64, H=32, G=8, D=128, seen=9000, dtype="bf16"),
        # one token for one user with a long document behind it
        dict(name="step_long", kind="step", B=1, H=32, G=4, D=128, seen=262000, dtype="fp16"),
        # five drafted tokens of 16 users, checked in one call
        dict(name="attn_draft", kind="attn", B=16, T=5, H=16, G=2, D=64, seen=6000, dtype="fp16",
             ragged=True),
        # a piece of a long prompt against what came before it
        dict(name="attn_chunk", kind="attn", B=1, T=2048, H=32, G=8, D=128, seen=30001,
             dtype="bf16", ragged=False),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_COST = {  # the most that a drawn case of each kind may take: bytes, operations
    "rope": (5e8, 1e11), "append": (2e8, 1e11), "read": (7e8, 1e11), "step": (6e8, 1e11),
    "attn": (3e8, 1e12)}


def draw(rng):
    kind = rng.choice(["rope", "rope", "rope", "append", "append", "read", "attn", "attn", "attn",
                       "step", "step", "step"])
    wide, half = ["bf16", "bf16", "fp16", "fp32"], ["bf16", "bf16", "fp16"]
    while True:
        c = dict(kind=kind, dtype=rng.choice(wide if kind in ("rope", "read") else half))
        G = _log(rng, 1, 16)
        H = G * rng.choice([1, 1, 2, 4, 5, 8])
        if kind == "rope":
            D = rng.choice([32, 64, 128, 64, 128, 80, 96, 2 * rng.randint(1, 128)])
            c.update(B=_log(rng, 1, 64), T=_log(rng, 1, 32768), H=H, G=G, D=D,
                     rot=rng.choice([D, D, 2 * max(1, D // 4), 2 * rng.randint(1, D // 2)]),
                     layout=rng.choice(["half", "interleaved"]), scale=rng.choice([1.0, 1.0, 1.25]),
                     positions=rng.choice(["none", "row", "token"]), seen=_log(rng, 1, 1000000),
                     train=rng.random() < 0.6)
        else:
            D = rng.choice([64, 128, 64, 128, 16 * rng.randint(1, 8)])
            c.update(B=_log(rng, 1, 64), G=G, D=D)
            if kind == "append":
                c.update(T=_log(rng, 1, 8192), seen=rng.choice([0, _log(rng, 1, 8192)]),
                         ragged=rng.random() < 0.5)
            elif kind == "read":
                seen = _log(rng, 1, 65536)
                start = rng.choice([0, rng.randint(0, seen - 1)])
                c.update(seen=seen, start=start, n=_log(rng, 1, seen - start))
            elif kind == "attn":
                c.update(T=_log(rng, 1, 4096), H=H, seen=rng.choice([0, _log(rng, 1, 32768)]),
                         ragged=rng.random() < 0.4)
            else:
                c.update(H=H, seen=_log(rng, 1, 262144))
        w = work(c)
        if w["bytes"] > _COST[kind][0] or w["flops"] > _COST[kind][1]:
            continue
        if kind == "attn" and c["B"] * c["H"] * c["T"] * _capacity(c) > 2 ** 31:
            continue                        # the plain form keeps the scores
        if kind != "rope" and c["B"] * c["G"] * _capacity(c) * c["D"] > 2 ** 30:
            continue
        return c


def _lengths(c):
    """New tokens of each row: the first has all T, the last about half."""
    B, T = c["B"], c["T"]
    return [T - b * T // (2 * B) if c.get("ragged") else T for b in range(B)]


def _seen(c):
    """Tokens that each row has in its cache before the call."""
    return [(b + 1) * c["seen"] // c["B"] for b in range(c["B"])]


def _new(c):
    return c.get("T", 0 if c["kind"] == "read" else 1)


def _capacity(c):
    """Slots a row: for what was there and the new tokens, and a block for what comes."""
    return (c["seen"] + _new(c) + 2 * BLOCK - 1) // BLOCK * BLOCK + BLOCK


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
class _Make:
    """Seeded tensors on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(DEV).manual_seed(seed)

    def normal(self, *shape, dtype=torch.float32, scale=1.0):
        return torch.randn(*shape, generator=self.gen, device=DEV).mul_(scale).to(dtype)

    def keys(self, *shape, dtype):
        """[.., tokens, heads or not, D]: channels of several widths, some off centre."""
        wide = torch.randn(shape[-1], generator=self.gen, device=DEV).mul_(0.5).exp_()
        off = torch.randn(shape[-1], generator=self.gen, device=DEV).mul_(0.5)
        return self.normal(*shape).mul_(wide).add_(off).to(dtype)

    def cache(self, B, G, slots, D):
        """Codes and scales of a cache whose every slot was written, in pieces of rows."""
        codes = torch.empty(B, G, slots, D, dtype=E4M3, device=DEV)
        scale = torch.empty(B, G, slots // BLOCK, device=DEV)
        wide = torch.randn(G, 1, D, generator=self.gen, device=DEV).mul_(0.5).exp_()
        for b in range(B):
            x = self.normal(G, slots, D).mul_(wide).view(G, -1, BLOCK, D)
            s = _power(_exponent(x.abs().amax((-1, -2)), "bf16"))
            codes[b] = (x / s[..., None, None]).to(E4M3).view(G, slots, D)
            scale[b] = s
        return codes, scale


def prepare(case, seed):
    c, m = case, _Make(seed)
    s, x = dict(case=dict(c)), {}
    dt, B, G, D, kind = DTYPES[c["dtype"]], c["B"], c["G"], c["D"], c["kind"]
    if kind == "rope":
        T, H = c["T"], c["H"]
        x["q"], x["k"] = (m.normal(B, T, n, D, dtype=dt) for n in (H, G))
        i = torch.arange(c["rot"] // 2, dtype=torch.float64, device=DEV)
        s["freqs"] = 10000.0 ** (-2 * i / c["rot"])
        first = torch.tensor(_seen(c), dtype=torch.int64, device=DEV)
        if c["positions"] == "row":          # of the row's first token
            s["positions"] = first
        elif c["positions"] == "token":      # documents behind one another
            t = torch.arange(T, device=DEV)
            s["positions"] = first[:, None] + t % random.Random(seed).randint(64, 4096)
        if c["train"]:
            s["dq"], s["dk"] = (m.normal(B, T, n, D, dtype=dt) for n in (H, G))
            for t in x.values():
                t.requires_grad_()
    else:
        slots = _capacity(c)
        for n in "kv":
            s["c" + n], s["s" + n] = m.cache(B, G, slots, D)
        s["seen"] = torch.tensor(_seen(c), dtype=torch.int32, device=DEV)
        s["counts"] = s["seen"].clone()
        new = ((B, c["T"]) if kind in ("append", "attn") else (B,))
        if kind in ("append", "step"):
            x["k"], x["v"] = m.keys(*new, G, D, dtype=dt), m.normal(*new, G, D, dtype=dt)
        if kind in ("attn", "step"):
            x["q"] = m.normal(*new, c["H"], D, dtype=dt)
        if kind == "attn":                   # the new tokens are in the cache already
            s["counts"] += torch.tensor(_lengths(c), dtype=torch.int32, device=DEV)
        if c.get("ragged"):
            s["lengths"] = torch.tensor(_lengths(c), dtype=torch.int32, device=DEV)
    s["x"] = x
    return s


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def _ours():
    """The package's entry points."""
    root = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..")
    sys.path.insert(0, os.path.join(root, "log-linear-attention_amd"))
    from hattention import quant_cache_apis, rotary_apis
    return rotary_apis, quant_cache_apis


_apis = None


def run(state):
    global _apis
    c, x, s = state["case"], state["x"], state
    kind = c["kind"]
    if own:
        if _apis is None:
            _apis = _ours()
        rope, qc = _apis
    if kind == "rope":
        f = rope.rotary_embedding if own else _plain_rope
        with torch.set_grad_enabled(bool(c["train"])):
            q, k = f(x["q"], x["k"], s["freqs"], s.get("positions"), c["layout"], c["scale"])
        if not c["train"]:
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad([q, k], [x["q"], x["k"]], [s["dq"], s["dk"]])
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    if own:
        cache = qc.QuantCache(s["ck"], s["cv"], s["sk"], s["sv"], s["counts"])
    if kind in ("append", "step"):
        s["counts"].copy_(s["seen"])
    if kind == "read":
        if own:
            k, v = qc.quant_cache_read(cache, DTYPES[c["dtype"]], c["start"], c["start"] + c["n"])
        else:
            k, v = _plain_read(s, c)
        return {"k": k, "v": v}
    if kind == "attn":
        if own:
            return {"o": qc.quant_cache_attention(cache, x["q"], lengths=s.get("lengths"))}
        return {"o": _plain_attn(s, x["q"], s.get("lengths"))}
    out = {"k": s["ck"], "v": s["cv"], "k_scale": s["sk"], "v_scale": s["sv"],
           "counts": s["counts"]}
    if kind == "append":
        if own:
            qc.quant_cache_append(cache, x["k"], x["v"], lengths=s.get("lengths"))
        else:
            _plain_append(s, x["k"], x["v"], s.get("lengths"))
        return out
    if own:
        o, cache = qc.quant_cache_step(cache, x["q"], x["k"], x["v"])
    else:
        _plain_append(s, x["k"][:, None], x["v"][:, None], None)
        o = _plain_attn(s, x["q"][:, None], None)[:, 0]
    return {"o": o, **out}


# --------------------------------------------------------------------------
# the plain forms
# --------------------------------------------------------------------------
def _plain_rope(q, k, freqs, positions, layout, scale):
    """Angles in 64 bits, sines and products in 32."""
    B, T = q.shape[:2]
    p = torch.arange(T, device=DEV).expand(B, T)
    if positions is not None:
        p = positions if positions.dim() == 2 else positions[:, None] + p
    angle = (p.double()[..., None] * freqs)[:, :, None]                  # [B, T, 1, rot / 2]
    cos, sin = ((f(angle) * scale).float() for f in (torch.cos, torch.sin))
    n = freqs.shape[0]

    def turn(x):
        f = x.float()
        r = f[..., :2 * n]
        a, b = (r[..., :n], r[..., n:]) if layout == "half" else (r[..., 0::2], r[..., 1::2])
        y = (a * cos - b * sin, a * sin + b * cos)
        y = torch.cat(y, -1) if layout == "half" else torch.stack(y, -1).flatten(-2)
        return torch.cat([y, f[..., 2 * n:]], -1).to(x.dtype)
    return turn(q), turn(k)


def _exponent(amax, dtype):
    """The least e with amax <= 448 * 2 ** e (448 = 0.875 * 2 ** 9), in its range."""
    m, x = torch.frexp(amax)
    e = x - 9 + (m > 0.875)
    return torch.where(amax > 0, e, LEAST).clamp(LEAST, MOST[dtype])


def _power(e):
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _plain_append(s, k, v, lengths):
    """Every block that a new token enters, made again: its old codes under the new scale
    where that grew, and the codes of the new tokens."""
    B, T, G, D = k.shape
    dtype = "fp16" if k.dtype == torch.float16 else "bf16"
    n0 = s["counts"].long()
    end = n0 + (lengths.long() if lengths is not None else T)
    blocks = (T + BLOCK - 2) // BLOCK + 1
    b0 = n0 // BLOCK
    at = b0[:, None] * BLOCK + torch.arange(blocks * BLOCK, device=DEV)  # [B, slots]
    bat = b0[:, None] + torch.arange(blocks, device=DEV)
    # a call's last blocks may lie past the cache of a row: they hold no token
    inside = (at < s["ck"].shape[2])[:, None, :, None]
    at, bat = at.clamp_max(s["ck"].shape[2] - 1), bat.clamp_max(s["sk"].shape[2] - 1)
    rows = torch.arange(B, device=DEV)[:, None]
    token = (at - n0[:, None]).clamp(0, T - 1)
    heads = torch.arange(G, device=DEV)[:, None]
    old = (at < n0[:, None])[:, None, :, None] & inside                  # [B, 1, slots, 1]
    new = ((at >= n0[:, None]) & (at < end[:, None]))[:, None, :, None] & inside
    for x, codes, scale in ((k, s["ck"], s["sk"]), (v, s["cv"], s["sv"])):
        had = codes[rows[..., None], heads, at[:, None]].float()        # [B, G, slots, D]
        was = scale[rows[..., None], heads, bat[:, None]]               # [B, G, blocks]
        y = x.float()[rows, token].transpose(1, 2)
        amax = torch.where(new, y, 0).abs().reshape(B, G, blocks, -1).amax(-1)
        e = _exponent(amax, dtype)
        some_old = old.view(B, 1, blocks, BLOCK).any(-1)
        some_new = new.view(B, 1, blocks, BLOCK).any(-1)
        now = torch.where(some_old, torch.maximum(_power(e), was), _power(e))
        now = torch.where(some_new, now, was)
        wide = lambda t: t.repeat_interleave(BLOCK, -1)[..., None]
        got = torch.where(new, (y / wide(now)).clamp(-448, 448),
                          torch.where(old, had * wide(was / now), had))
        codes[rows[..., None], heads, at[:, None]] = got.to(E4M3)
        scale[rows[..., None], heads, bat[:, None]] = now
    s["counts"].copy_(end)


def _values(codes, scale):
    B, G, slots, D = codes.shape
    return codes.float().view(B, G, -1, BLOCK, D) * scale[..., None, None]


def _plain_read(s, c):
    lo, hi = c["start"], c["start"] + c["n"]
    held = (torch.arange(lo, hi, device=DEV) < s["counts"][:, None])[..., None, None]
    return [torch.where(held, _values(s["c" + n], s["s" + n]).flatten(2, 3)[:, :, lo:hi]
                        .transpose(1, 2), 0).to(DTYPES[c["dtype"]]) for n in "kv"]


def _plain_attn(s, q, lengths):
    """All of the cache's slots against all queries; those that a query does not see are
    taken out."""
    B, T, H, D = q.shape
    G = s["ck"].shape[1]
    k, v = (_values(s["c" + n], s["s" + n]).flatten(2, 3) for n in "kv")
    n = s["counts"].long()
    t = torch.arange(T, device=DEV)
    new = lengths.long() if lengths is not None else torch.full_like(n, T)
    last = torch.where(t < new[:, None], (n - new)[:, None] + t, -1)     # [B, T]
    seen = torch.arange(k.shape[2], device=DEV) <= last[..., None]
    seen = seen[:, None, None]                                           # [B, 1, 1, T, slots]
    x = (q.float() * D ** -0.5).view(B, T, G, H // G, D).permute(0, 2, 3, 1, 4)
    p = (x.reshape(B, G, -1, D) @ k.transpose(-1, -2)).view(B, G, H // G, T, -1)
    p = torch.where(seen, p, -1e30)
    p = torch.where(seen, (p - p.amax(-1, keepdim=True)).exp(), 0)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    o = (p.view(B, G, (H // G) * T, -1) @ v).view(B, G, H // G, T, D)
    return o.permute(0, 3, 1, 2, 4).reshape(B, T, H, D).to(q.dtype)


# --------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------
def work(case):
    c = case
    kind, B, G, D, e = c["kind"], c["B"], c["G"], c["D"], DTYPES[c["dtype"]].itemsize
    if kind == "rope":
        n = B * c["T"] * (c["H"] + c["G"])
        passes = 2 if c["train"] else 1
        return dict(bytes=2 * n * D * e * passes, flops=3 * n * c["rot"] * passes)
    if kind == "append":
        n = sum(_lengths(c)) * G * D
        return dict(bytes=2 * n * (e + 1), flops=4 * n)
    if kind == "read":
        held = sum(min(max(m - c["start"], 0), c["n"]) for m in _seen(c))
        return dict(bytes=2 * G * D * (held + B * c["n"] * e), flops=2 * G * D * held)
    T, H = _new(c), c["H"]
    new = _lengths(c) if kind == "attn" else [1] * B
    keys = sum(m + n for m, n in zip(_seen(c), new))
    pairs = sum(n * m + n * (n + 1) // 2 for m, n in zip(_seen(c), new))
    nbytes = 2 * keys * G * (D + 4 / BLOCK) + (sum(new) + B * T) * H * D * e
    if kind == "step":
        nbytes += 2 * B * G * D * (e + 1)
    return dict(bytes=nbytes, flops=4 * D * H * pairs)


# --------------------------------------------------------------------------
# the same results from the definitions, in 64 bits
# --------------------------------------------------------------------------
def exact(case, seed):
    c = case
    s = prepare(c, seed)
    x = {n: t.detach() for n, t in s["x"].items()}
    with torch.no_grad():
        if c["kind"] == "rope":
            return _exact_rope(c, s, x)
        if c["kind"] == "read":
            out = {}
            for n in "kv":
                y = torch.zeros(c["B"], c["n"], c["G"], c["D"], dtype=torch.float64, device=DEV)
                for b, m in enumerate(_seen(c)):
                    top = min(m, c["start"] + c["n"])
                    if top > c["start"]:
                        f = _exact_cache(s, n, b, top)[:, c["start"]:]
                        y[b, :top - c["start"]] = f.transpose(0, 1)
                out[n] = y
            return out
        out = {}
        if c["kind"] in ("append", "step"):
            for n in "kv":
                new = x[n] if c["kind"] == "append" else x[n][:, None]
                out[n], out[n + "_scale"] = _exact_append(c, s, n, new)
        if c["kind"] == "step":
            out["o"] = _exact_attn(c, x["q"][:, None], s, [m + 1 for m in _seen(c)], [1] * c["B"],
                                   out)[:, 0]
        if c["kind"] == "attn":
            new = _lengths(c)
            out["o"] = _exact_attn(c, x["q"], s, [m + n for m, n in zip(_seen(c), new)], new)
        return out


def _exact_rope(c, s, x):
    """Each pair as one complex number, times the unit number of its angle."""
    B, T, r = c["B"], c["T"], c["rot"]
    p = s.get("positions")
    t = torch.arange(T, device=DEV, dtype=torch.float64)
    p = t.repeat(B, 1) if p is None else p.double() if p.dim() == 2 else t + p.double()[:, None]
    unit = torch.polar(torch.full_like(p, c["scale"])[..., None].expand(B, T, r // 2).contiguous(),
                       p[..., None] * s["freqs"])[:, :, None]
    if c["layout"] == "half":
        first, second = slice(0, r // 2), slice(r // 2, r)
    else:
        first, second = slice(0, r, 2), slice(1, r, 2)

    def turned(z, by):
        y = z.double()
        w = torch.complex(y[..., first].clone(), y[..., second].clone()) * by
        y[..., first], y[..., second] = w.real, w.imag
        return y
    out = {n: turned(x[n], unit) for n in "qk"}
    if c["train"]:
        out.update({"d" + n: turned(s["d" + n], unit.conj()) for n in "qk"})
    return out


def _exact_round(y):
    """To the nearest of the numbers of 4 bits from 2 ** -6 on, steps of 2 ** -9 below; ties
    to even; at most 448."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6)) + 1e-9) - 3)
    return (torch.round(y / step) * step).clamp(-448.0, 448.0)


def _exact_append(c, s, n, new):
    """Codes and scales of one of k and v after the call, block by block of each row."""
    codes, scale = s["c" + n].double(), s["s" + n].double()
    for b, (m, k) in enumerate(zip(_seen(c), _lengths(c) if "T" in c else [1] * c["B"])):
        at = m
        while at < m + k:
            j, top = at // BLOCK, min((at // BLOCK + 1) * BLOCK, m + k)
            y = new[b, at - m:top - m].double().transpose(0, 1)          # [G, tokens, D]
            # -inf for a block of zeros; a power of two is itself
            e = torch.ceil(torch.log2(y.abs().amax((1, 2)) / 448.0) - 1e-9)
            now = torch.exp2(e.clamp(LEAST, MOST[c["dtype"]]))
            if at > j * BLOCK:
                now = torch.maximum(now, scale[b, :, j])
                was = codes[b, :, j * BLOCK:at]
                codes[b, :, j * BLOCK:at] = _exact_round(was * (scale[b, :, j] / now)[:, None, None])
            codes[b, :, at:top] = _exact_round(y / now[:, None, None])
            scale[b, :, j] = now
            at = top
    return codes, scale


def _exact_cache(s, n, b, top, new=None):
    codes, scale = (new[n][b], new[n + "_scale"][b]) if new else (s["c" + n][b], s["s" + n][b])
    blocks = -(-top // BLOCK)
    y = codes[:, :blocks * BLOCK].double() * \
        scale[:, :blocks].double().repeat_interleave(BLOCK, 1)[..., None]
    return y[:, :top]


def _exact_attn(c, q, s, counts, lens, new=None):
    """Head by head; query t of a row's `lens` new tokens is at counts - lens + t."""
    H, G, D = c["H"], c["G"], c["D"]
    o = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    for b, (n, m) in enumerate(zip(counts, lens)):
        k, v = (_exact_cache(s, w, b, n, new) for w in "kv")
        hidden = torch.arange(n, device=DEV) > (n - m + torch.arange(m, device=DEV))[:, None]
        for h in range(H):
            z = q[b, :m, h].double() @ k[h // (H // G)].T / math.sqrt(D)
            o[b, :m, h] = torch.softmax(z.masked_fill_(hidden, -math.inf), 1) @ v[h // (H // G)]
    return o
