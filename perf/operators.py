"""The block operators around the attention core, measured case by case: layer norm (forward and
backward), linear layers in 8-bit integers, rotary positions with several axes.

Every case runs in two forms on the same state.  With ``own`` false, ``run`` computes the operator from
elementary torch operations in 32 bits (64 where 32 would lose what matters) and rounds once at the end;
with ``own`` true it makes the calls of ``ppdl`` that a program makes.  ``exact`` evaluates the operators'
definitions in 64 bits, apart from both.
"""
import functools
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


@functools.lru_cache(maxsize=1)
def _ppdl():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ppdoclayout-ggml_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import ppdl
    return ppdl


# ---- cases ---------------------------------------------------------------------------------------

def listed():
    return [
        # one token of a decoder being served: latency alone
        {"name": "ln one token", "op": "ln", "rows": 1, "dim": 4096, "type": "bf16", "wtype": "bf16", "residual": True, "stats": False},
        # the memory tokens of four pages (13125 each), 256 wide, with the residual added on the way
        {"name": "ln memory tokens", "op": "ln", "rows": 52500, "dim": 256, "type": "f32", "wtype": "f32", "residual": True, "stats": True},
        # the 300 queries of eight pages in training
        {"name": "ln bwd queries", "op": "ln_bwd", "rows": 2400, "dim": 256, "type": "f32", "wtype": "f32", "residual": True},
        # a training batch of a wide model, weights kept in 32 bits
        {"name": "ln bwd wide", "op": "ln_bwd", "rows": 16384, "dim": 4096, "type": "bf16", "wtype": "f32", "residual": False},
        # rows whose length is odd, so that no two of them start on the same alignment
        {"name": "ln bwd odd rows", "op": "ln_bwd", "rows": 4099, "dim": 1153, "type": "f16", "wtype": "f16", "residual": False},
        # one token through a square projection: the weights' bytes are the bound
        {"name": "linear one token", "op": "linear", "m": 1, "k": 4096, "n": 4096, "type": "bf16", "act": "none", "bias": False, "residual": False},
        # the feed-forward expansion of the decoder, eight pages of 300 queries
        {"name": "linear decoder ffn", "op": "linear", "m": 2400, "k": 256, "n": 1024, "type": "f32", "act": "relu", "bias": True, "residual": False},
        # the six stacked value projections over the memory tokens of four pages
        {"name": "linear value projections", "op": "linear", "m": 52500, "k": 256, "n": 1536, "type": "f32", "act": "none", "bias": True, "residual": False},
        # sizes that divide by nothing
        {"name": "linear odd sizes", "op": "linear", "m": 777, "k": 1111, "n": 2047, "type": "f16", "act": "gelu", "bias": True, "residual": True},
        # a prefill of a large model: the integer rate is the bound
        {"name": "linear prefill", "op": "linear", "m": 8192, "k": 8192, "n": 8192, "type": "bf16", "act": "none", "bias": False, "residual": False},
        # one new token for each of 64 sequences, eight key heads shared by 32 query heads
        {"name": "rotary new tokens", "op": "rotary", "batch": 64, "length": 1, "qheads": 32, "kheads": 8, "dim": 128, "rotated": 128, "s0": 16, "s1": 24, "s2": 24, "far": 32768, "type": "bf16", "paired": False, "inverse": False},
        # the gradient of the queries and keys of eight frames of 50 x 50 patches
        {"name": "rotary bwd patches", "op": "rotary", "batch": 8, "length": 2500, "qheads": 16, "kheads": 16, "dim": 64, "rotated": 64, "s0": 8, "s1": 12, "s2": 12, "far": 2500, "type": "f32", "paired": False, "inverse": True},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm, odd as often as even."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["ln", "ln_bwd", "linear", "linear", "rotary"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op in ("ln", "ln_bwd"):
        dim = rng.choice([_spread(rng, 8, 16384), 8 * _spread(rng, 1, 2048)])
        rows = _spread(rng, 1, max(1, min(400000, 60000000 // dim)))
        case = {"op": op, "rows": rows, "dim": dim, "type": kind, "wtype": rng.choice([kind, "f32"]), "residual": rng.random() < 0.5}
        if op == "ln":
            case["stats"] = rng.random() < 0.5
        return case
    if op == "linear":
        k = rng.choice([_spread(rng, 16, 12000), 64 * _spread(rng, 1, 128)])
        n = rng.choice([_spread(rng, 16, 12000), 64 * _spread(rng, 1, 128)])
        # at most a fifth of the largest listed product, and outputs that fit easily
        m = _spread(rng, 1, max(1, min(60000, int(1e11) // (k * n), 200000000 // n, 200000000 // k)))
        return {"op": op, "m": m, "k": k, "n": n, "type": kind, "act": rng.choice(["none", "relu", "silu", "gelu"]), "bias": rng.random() < 0.5, "residual": rng.random() < 0.3}
    dim = rng.choice([32, 64, 96, 128, 256])
    rotated = rng.choice([dim, dim, dim // 2])
    pairs = rotated // 2
    s0 = rng.randint(0, pairs)
    s1 = rng.randint(0, pairs - s0)
    kheads = rng.choice([1, 2, 4, 8])
    qheads = kheads * rng.choice([1, 2, 4, 7])
    batch = _spread(rng, 1, 64)
    length = _spread(rng, 1, max(1, min(16384, 40000000 // (batch * (qheads + kheads) * dim))))
    return {"op": op, "batch": batch, "length": length, "qheads": qheads, "kheads": kheads, "dim": dim, "rotated": rotated, "s0": s0, "s1": s1, "s2": pairs - s0 - s1,
            "far": _spread(rng, 64, 1000000), "type": kind, "paired": rng.random() < 0.5, "inverse": rng.random() < 0.5}


# ---- what a program has in hand ------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPES[case["type"]]

    def normal(*shape, scale=1.0, shift=0.0, to=t):
        return torch.randn(shape, generator=g, device="cuda").mul_(scale).add_(shift).to(to)

    st = {"case": case}
    if case["op"] in ("ln", "ln_bwd"):
        rows, dim, wt = case["rows"], case["dim"], DTYPES[case["wtype"]]
        st["weight"] = normal(dim, scale=0.2, shift=1.0, to=wt)
        st["bias"] = normal(dim, scale=0.2, to=wt)
        if case["op"] == "ln":
            st["x"] = normal(rows, dim, scale=1.5, shift=0.3)
            st["residual"] = normal(rows, dim) if case["residual"] else None
        else:
            # what the forward pass kept: its input and each row's statistics
            st["x"] = normal(rows, dim, scale=1.5, shift=0.3)
            x = st["x"].double()
            st["mean"] = x.mean(1).float()
            st["rstd"] = (x.var(1, unbiased=False) + 1e-5).rsqrt().float()
            st["dy"] = normal(rows, dim, scale=0.1)
            st["dsum"] = normal(rows, dim, scale=0.1) if case["residual"] else None
    elif case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        st["x"] = normal(m, k)
        # weights quantised once at load, channel by channel, rows on 16-byte strides
        w = torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)
        st["wscale"] = w.abs().amax(1) / 127.0
        st["weight"] = torch.zeros(n, (k + 15) // 16 * 16, dtype=torch.int8, device="cuda")[:, :k]
        st["weight"].copy_((w / st["wscale"][:, None]).round().clamp_(-127, 127))
        st["bias"] = normal(n, scale=0.1, to=torch.float32) if case["bias"] else None
        st["residual"] = normal(m, n) if case["residual"] else None
    else:
        b, length, d = case["batch"], case["length"], case["dim"]
        # queries and keys side by side in rows of one projection's output
        qk = normal(b, length, case["qheads"] + case["kheads"], d)
        st["q"], st["k"] = qk[:, :, :case["qheads"]], qk[:, :, case["qheads"]:]
        st["positions"] = torch.randint(0, case["far"], (3, b, length), generator=g, device="cuda")
        pairs = case["rotated"] // 2
        st["freq"] = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs)
        st["sections"] = (case["s0"], case["s1"], case["s2"])
        # which axis turns each pair
        st["axis"] = torch.tensor([a for a, s in enumerate(st["sections"]) for _ in range(s)], device="cuda")
    return st


# ---- one pass ------------------------------------------------------------------------------------

def _ln(st):
    case, x = st["case"], st["x"]
    if own:
        return _ppdl().layernorm(x, st["weight"], st["bias"], 1e-5, residual=st["residual"], return_sum=case["residual"], return_stats=case["stats"])
    s = x if st["residual"] is None else (x.float() + st["residual"].float()).to(x.dtype)
    f = s.float()
    mean = f.mean(1, keepdim=True)
    c = f - mean
    rstd = torch.rsqrt((c * c).mean(1, keepdim=True) + 1e-5)
    out = ((c * rstd * st["weight"].float() + st["bias"].float()).to(x.dtype),)
    out += (s,) if case["residual"] else ()
    out += (mean[:, 0], rstd[:, 0]) if case["stats"] else ()
    return out if len(out) > 1 else out[0]


def _ln_bwd(st):
    x, wt = st["x"], st["weight"].dtype
    if own:
        return _ppdl().layernorm_backward(st["dy"], x, st["weight"], st["mean"], st["rstd"], dsum=st["dsum"])
    dy = st["dy"].float()
    xh = (x.float() - st["mean"][:, None]) * st["rstd"][:, None]
    wdy = dy * st["weight"].float()
    dx = (wdy - wdy.mean(1, keepdim=True) - xh * (wdy * xh).mean(1, keepdim=True)) * st["rstd"][:, None]
    if st["dsum"] is not None:
        dx = dx + st["dsum"].float()
    return dx.to(x.dtype), (dy * xh).sum(0).to(wt), dy.sum(0).to(wt)


def _linear(st):
    case, x = st["case"], st["x"]
    if own:
        return _ppdl().linear_i8(x, st["weight"], st["wscale"], bias=st["bias"], act=case["act"], residual=st["residual"])
    xf = x.float()
    # 64 bits decide the scale's last bit and the values next to a half; whole products of 127 x 127 stay exact in 32 bits up to 1040 of them
    scale = (xf.abs().amax(1, keepdim=True).double() / 127.0).float()
    q = (xf.double() / scale.double()).round().nan_to_num(0.0)
    t = torch.float32 if case["k"] <= 1040 else torch.float64
    y = (q.to(t) @ st["weight"].to(t).t()).float() * scale * st["wscale"]
    if st["bias"] is not None:
        y = y + st["bias"]
    if case["act"] == "relu":
        y = y.clamp_min(0.0)
    elif case["act"] == "silu":
        y = y / (1.0 + torch.exp(-y))
    elif case["act"] == "gelu":
        y = 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    if st["residual"] is not None:
        y = y + st["residual"].float()
    return y.to(x.dtype)


def _rotated(x, c, s, rotated, paired):
    """The first `rotated` values of each head turned pair by pair, the others as they are."""
    f = x.float()
    r = f[..., :rotated]
    a, b = (r[..., 0::2], r[..., 1::2]) if paired else (r[..., :rotated // 2], r[..., rotated // 2:])
    u, v = a * c - b * s, b * c + a * s
    r = torch.stack((u, v), -1).flatten(-2) if paired else torch.cat((u, v), -1)
    return torch.cat((r, f[..., rotated:]), -1).to(x.dtype)


def _rotary(st):
    case = st["case"]
    if own:
        return _ppdl().rotary(st["q"], st["k"], st["positions"], st["freq"], st["sections"], interleaved=case["paired"], inverse=case["inverse"])
    angle = st["positions"][st["axis"]].permute(1, 2, 0).double() * st["freq"]
    c, s = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]
    if case["inverse"]:
        s = -s
    return tuple(_rotated(x, c, s, case["rotated"], case["paired"]) for x in (st["q"], st["k"]))


def run(state):
    return {"ln": _ln, "ln_bwd": _ln_bwd, "linear": _linear, "rotary": _rotary}[state["case"]["op"]](state)


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    e = SIZE[case["type"]]
    if case["op"] in ("ln", "ln_bwd"):
        n, w = case["rows"] * case["dim"], case["dim"] * SIZE[case["wtype"]]
        if case["op"] == "ln":
            return {"bytes": n * e * (4 if case["residual"] else 2) + 2 * w + (8 * case["rows"] if case["stats"] else 0), "flops": 8 * n}
        return {"bytes": n * e * (4 if case["residual"] else 3) + 8 * case["rows"] + 3 * w, "flops": 14 * n}
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": m * k * e + n * k + 4 * n + m * n * e * (2 if case["residual"] else 1) + (4 * n if case["bias"] else 0), "flops": 2 * m * k * n}
    n = case["batch"] * case["length"]
    values = n * (case["qheads"] + case["kheads"]) * case["dim"]
    return {"bytes": 2 * values * e + 3 * 8 * n + 4 * case["rotated"], "flops": 3 * values}


# ---- the definitions in 64 bits ------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "ln":
        x, out = st["x"].double(), ()
        if case["residual"]:
            # the sum is a value of its type: the norm is of what is stored
            x = (x + st["residual"].double()).to(st["x"].dtype).double()
            out = (x,)
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        sd = torch.sqrt(var + 1e-5)
        y = st["bias"].double() + st["weight"].double() * ((x - mean) / sd)
        out = (y,) + out + ((mean.squeeze(1), 1.0 / sd.squeeze(1)) if case["stats"] else ())
        return out if len(out) > 1 else y
    if case["op"] == "ln_bwd":
        # through the Jacobian's two projections: on the constants and on the normalised row
        dy, d = st["dy"].double(), case["dim"]
        r = st["rstd"].double().unsqueeze(1)
        xh = torch.addcmul(-st["mean"].double().unsqueeze(1) * r, st["x"].double(), r)
        g = dy * st["weight"].double()
        along = torch.einsum("rd,rd->r", g, xh).unsqueeze(1) / d
        dx = r * (g - g.sum(1, keepdim=True) / d - along * xh)
        if case["residual"]:
            dx += st["dsum"].double()
        return dx, torch.einsum("rd,rd->d", dy, xh), torch.einsum("rd->d", dy)
    if case["op"] == "linear":
        x = st["x"].double()
        # the scale is a 32-bit number: the nearest to a 127th of the row's largest value
        step = (x.abs().max(dim=1).values / 127).float().double()
        q = torch.where(step.unsqueeze(1) > 0, torch.round(x / step.unsqueeze(1)), torch.zeros_like(x))
        y = torch.einsum("mk,nk->mn", q, st["weight"].double())
        y *= step.unsqueeze(1)
        y *= st["wscale"].double()
        if case["bias"]:
            y += st["bias"].double()
        if case["act"] == "relu":
            y = torch.maximum(y, torch.zeros_like(y))
        elif case["act"] == "silu":
            y = y * torch.sigmoid(y)
        elif case["act"] == "gelu":
            y = y * torch.special.ndtr(y)
        return y + st["residual"].double() if case["residual"] else y
    # a pair is one complex number, turned by its own position times its own frequency
    sign = -1.0 if case["inverse"] else 1.0
    at = torch.cat([st["positions"][a].unsqueeze(-1).expand(-1, -1, s) for a, s in enumerate(st["sections"])], -1)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), sign * at.double() * st["freq"]).unsqueeze(2)
    half, out = case["rotated"] // 2, []
    for x in (st["q"], st["k"]):
        y = x.double()
        pair = y[..., :2 * half].unflatten(-1, (half, 2)) if case["paired"] else y[..., :2 * half].unflatten(-1, (2, half)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        z = z if case["paired"] else z.transpose(-1, -2)
        out.append(torch.cat((z.flatten(-2), y[..., 2 * half:]), -1))
    return tuple(out)
