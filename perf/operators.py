"""Measured cases of the language-model operators: the residual RMS norm and the gated feed-forward block.

`run` computes a case either in plain torch operations (32 bits, one rounding at the end) or, with `own` set, through
`framepack_amd.ops`; `exact` computes it from the definitions in 64 bits.

  norm      h = resid + x,  y = h / sqrt(mean(h^2) + eps) * weight
  norm8     the same with y in e4m3 and one scale a row: scale = max|y| / 448, y ~ scale * q
  norm_grad from dy and the gradient dh that reaches h by its other path: dx (which is dresid too) and dweight
  ff        h = act(x . Wg^T + bg) * (x . Wu^T + bu); with keep, also both projections as a backward pass needs them
  ff8       the same on e4m3 operands with a scale a row of x and a scale a row of Wg and Wu
  ff_grad   from dh and the kept projections: dx, dWg, dWu (and the biases' gradients)
"""
import math

import torch

own = False

EPS = 1e-6
FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ---- cases -----------------------------------------------------------------------------------------------------

def listed():
    return [
        # one token of a decoding step through a norm of the text encoder's width: latency alone
        dict(name="norm, one token", op="norm", dtype="bf16", rows=1, cols=4096),
        # the vision tower's 27 x 27 patches, a width that is no power of two, half precision
        dict(name="norm, vision patches", op="norm", dtype="f16", rows=729, cols=1152),
        # the longest ordinary sequence (the packed video tokens of a section) at the text encoder's width: bandwidth
        dict(name="norm, long sequence", op="norm", dtype="bf16", rows=19385, cols=4096),
        # a text prompt on its way into 8-bit linears
        dict(name="norm to 8 bits, prompt", op="norm8", dtype="bf16", rows=512, cols=4096),
        # a training batch with a ragged row count
        dict(name="norm gradient, batch", op="norm_grad", dtype="bf16", rows=8191, cols=4096),
        # one decoded token: both weight matrices are read once, nothing is reused
        dict(name="ff, one token", op="ff", dtype="bf16", act="silu", bias=False, keep=False, rows=1, cols=4096, inner=14336),
        # a small decoding batch on 8-bit weights
        dict(name="ff in 8 bits, 16 tokens", op="ff8", dtype="bf16", act="silu", bias=False, rows=16, cols=4096, inner=14336),
        # vision patches, gated tanh-GELU with biases, projections kept for training; ragged rows and a width off the tiles
        dict(name="ff, vision patches", op="ff", dtype="f16", act="gelu", bias=True, keep=True, rows=729, cols=1152, inner=4304),
        # a batch of prompts on 8-bit weights
        dict(name="ff in 8 bits, prompts", op="ff8", dtype="bf16", act="silu", bias=False, rows=4096, cols=4096, inner=14336),
        # the longest sequence: all matrix work
        dict(name="ff, long sequence", op="ff", dtype="bf16", act="silu", bias=False, keep=False, rows=19385, cols=4096, inner=14336),
        # the vision block's gradients
        dict(name="ff gradient, vision", op="ff_grad", dtype="f16", act="gelu", bias=True, rows=729, cols=1152, inner=4304),
        # a training batch's gradients
        dict(name="ff gradient, batch", op="ff_grad", dtype="bf16", act="silu", bias=False, rows=4096, cols=4096, inner=11008),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm8", "norm_grad", "ff", "ff8", "ff_grad"])
    case = dict(op=op, dtype=rng.choice(["bf16", "bf16", "f16"]), rows=_log(rng, 1, 19385))
    if op.startswith("norm"):
        # any width; three in four are multiples of 8, as widths mostly are
        case["cols"] = _log(rng, 64, 8192) if rng.random() < 0.25 else 8 * _log(rng, 8, 1024)
        if op == "norm8":
            case["dtype"] = "bf16"
        return case
    case["act"] = rng.choice(["silu", "gelu"])
    case["bias"] = rng.random() < 0.3
    if op == "ff8":
        case["dtype"] = "bf16"
        case["cols"], case["inner"] = 128 * _log(rng, 1, 64), 8 * _log(rng, 8, 1792)
    else:
        case["cols"] = _log(rng, 64, 8192) if rng.random() < 0.25 else 64 * _log(rng, 1, 128)
        case["inner"] = _log(rng, 64, 14336) if rng.random() < 0.25 else 16 * _log(rng, 4, 896)
    if op == "ff":
        case["keep"] = rng.random() < 0.3
    most = 19385 * 4096 * 14336 // (4 if op == "ff_grad" else 1)
    case["rows"] = max(1, min(case["rows"], most // (case["cols"] * case["inner"])))
    return case


def work(case):
    op, r, c = case["op"], case["rows"], case["cols"]
    if op == "norm":
        return {"bytes": 8 * r * c + 2 * c, "flops": 6 * r * c}
    if op == "norm8":
        return {"bytes": 7 * r * c + 4 * r + 2 * c, "flops": 8 * r * c}
    if op == "norm_grad":
        return {"bytes": 8 * r * c + 4 * c, "flops": 14 * r * c}
    f = case["inner"]
    if op == "ff8":
        return {"bytes": r * c + 2 * f * c + 2 * r * f + 4 * r + 8 * f, "flops": 4 * r * c * f}
    if op == "ff":
        return {"bytes": 2 * r * c + 4 * f * c + 2 * r * f * (3 if case["keep"] else 1), "flops": 4 * r * c * f}
    return {"bytes": 4 * r * c + 8 * f * c + 6 * r * f, "flops": 8 * r * c * f}


# ---- inputs ----------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, r, c = TYPES[case["dtype"]], case["rows"], case["cols"]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * std

    if case["op"].startswith("norm"):
        weight = (1.0 + normal(c, std=0.2)).to(t)
        # a residual stream has a few channels that are far larger than the others
        big = 1.0 + 30.0 * (torch.rand(c, generator=g, device="cuda") < 0.004)
        live = torch.ones(r, 1, device="cuda")
        live[r - r // 16:] = 0                                        # padding behind the last token
        if case["op"] == "norm_grad":
            return dict(case, dy=(normal(r, c, std=0.01) * live).to(t), h=(normal(r, c, std=2.0) * big * live).to(t),
                        dh=(normal(r, c, std=0.01) * live).to(t), weight=weight)
        return dict(case, x=(normal(r, c) * live).to(t), resid=(normal(r, c, std=2.0) * big * live).to(t), weight=weight)

    f = case["inner"]
    s = dict(case, b_gate=None, b_up=None)
    x = normal(r, c)
    wg, wu = normal(f, c, std=c ** -0.5), normal(f, c, std=c ** -0.5)
    if case["bias"]:
        s["b_gate"], s["b_up"] = normal(f, std=0.1).to(t), normal(f, std=0.1).to(t)
    if case["op"] == "ff8":
        for key, v in (("x", x), ("w_gate", wg), ("w_up", wu)):
            scale = (v.abs().amax(dim=1) / FP8_MAX).clamp_min(1e-12)
            s[key], s[key + "_scale"] = (v / scale[:, None]).to(FP8), scale
        return s
    s["x"], s["w_gate"], s["w_up"] = x.to(t), wg.to(t), wu.to(t)
    if case["op"] == "ff_grad":
        s["dh"] = normal(r, f, std=0.01).to(t)
        s["gate"], s["up"] = normal(r, f).to(t), normal(r, f).to(t)   # as the forward pass kept them
    return s


# ---- one pass --------------------------------------------------------------------------------------------------

def _norm(s):
    if own:
        from framepack_amd import ops
        y, h = ops.rmsnorm_residual(s["x"], s["weight"], s["resid"], eps=EPS)
        return {"y": y, "h": h}
    h = s["x"].float() + s["resid"].float()
    y = h * torch.rsqrt(h.square().mean(dim=1, keepdim=True) + EPS) * s["weight"].float()
    return {"y": y.to(s["x"].dtype), "h": h.to(s["x"].dtype)}


def _norm8(s):
    if own:
        from framepack_amd import ops
        q, scale, h = ops.rmsnorm_residual_fp8(s["x"], s["weight"], s["resid"], eps=EPS)
        return {"q": q, "scale": scale, "h": h}
    h = s["x"].float() + s["resid"].float()
    y = h * torch.rsqrt(h.square().mean(dim=1, keepdim=True) + EPS) * s["weight"].float()
    amax = y.abs().amax(dim=1)
    scale = torch.where(amax > 0, amax / FP8_MAX, torch.ones_like(amax))
    return {"q": (y / scale[:, None]).to(FP8), "scale": scale, "h": h.to(s["x"].dtype)}


def _norm_grad(s):
    if own:
        from framepack_amd import ops
        dx, dweight = ops.rmsnorm_residual_backward(s["dy"], s["h"], s["weight"], dh=s["dh"], eps=EPS)
        return {"dx": dx, "dweight": dweight}
    h, dy = s["h"].float(), s["dy"].float()
    r = torch.rsqrt(h.square().mean(dim=1, keepdim=True) + EPS)
    n = h * r
    dn = dy * s["weight"].float()
    dx = s["dh"].float() + r * (dn - n * (dn * n).mean(dim=1, keepdim=True))
    return {"dx": dx.to(s["h"].dtype), "dweight": (dy * n).sum(dim=0).to(s["weight"].dtype)}


def _act(name, v):
    """act(v) and its derivative."""
    if name == "silu":
        e = torch.sigmoid(v)
        return v * e, e * (1 + v * (1 - e))
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (v + 0.044715 * v ** 3))
    return 0.5 * v * (1 + t), 0.5 * (1 + t) + 0.5 * v * (1 - t * t) * k * (1 + 3 * 0.044715 * v * v)


def _ff(s):
    if own:
        from framepack_amd import ops
        act = ops.ACT_SILU if s["act"] == "silu" else ops.ACT_GELU
        got = ops.gated_ff(s["x"], s["w_gate"], s["w_up"], s["b_gate"], s["b_up"], act=act, keep=s["keep"])
        return {"h": got[0], "gate": got[1], "up": got[2]} if s["keep"] else {"h": got}
    t, x = s["x"].dtype, s["x"].float()
    g, u = x @ s["w_gate"].float().t(), x @ s["w_up"].float().t()
    if s["bias"]:
        g, u = g + s["b_gate"].float(), u + s["b_up"].float()
    h = (_act(s["act"], g)[0] * u).to(t)
    return {"h": h, "gate": g.to(t), "up": u.to(t)} if s["keep"] else {"h": h}


def _ff8(s):
    if own:
        from framepack_amd import ops
        act = ops.ACT_SILU if s["act"] == "silu" else ops.ACT_GELU
        return {"h": ops.gated_ff_fp8(s["x"], s["x_scale"], s["w_gate"], s["w_gate_scale"], s["w_up"], s["w_up_scale"],
                                      s["b_gate"], s["b_up"], act=act)}
    x = s["x"].float() * s["x_scale"][:, None]
    g = x @ (s["w_gate"].float() * s["w_gate_scale"][:, None]).t()
    u = x @ (s["w_up"].float() * s["w_up_scale"][:, None]).t()
    if s["bias"]:
        g, u = g + s["b_gate"].float(), u + s["b_up"].float()
    return {"h": (_act(s["act"], g)[0] * u).to(torch.bfloat16)}


def _ff_grad(s):
    if own:
        from framepack_amd import ops
        act = ops.ACT_SILU if s["act"] == "silu" else ops.ACT_GELU
        dx, dwg, dwu, dbg, dbu = ops.gated_ff_backward(s["dh"], s["x"], s["w_gate"], s["w_up"], s["gate"], s["up"], act=act,
                                                       bias=s["bias"])
    else:
        t, dh = s["x"].dtype, s["dh"].float()
        a, da = _act(s["act"], s["gate"].float())
        dg, du = dh * s["up"].float() * da, dh * a
        dx = (dg @ s["w_gate"].float() + du @ s["w_up"].float()).to(t)
        dwg, dwu = (dg.t() @ s["x"].float()).to(t), (du.t() @ s["x"].float()).to(t)
        dbg, dbu = (dg.sum(dim=0).to(t), du.sum(dim=0).to(t)) if s["bias"] else (None, None)
    got = {"dx": dx, "dw_gate": dwg, "dw_up": dwu}
    return dict(got, db_gate=dbg, db_up=dbu) if s["bias"] else got


def run(state):
    return {"norm": _norm, "norm8": _norm8, "norm_grad": _norm_grad, "ff": _ff, "ff8": _ff8, "ff_grad": _ff_grad}[state["op"]](state)


# ---- from the definitions, in 64 bits -----------------------------------------------------------------------------

def _e4m3(v):
    """The nearest e4m3 values (ties to even) of |v| <= 448: 3 mantissa bits, steps of 2^-9 below 2^-6."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(v / step) * step


def exact(case, seed):
    s = {k: v.double() if torch.is_tensor(v) else v for k, v in prepare(case, seed).items()}
    op = case["op"]
    if op in ("norm", "norm8"):
        h = s["resid"] + s["x"]
        y = s["weight"] * h / torch.sqrt((h * h).sum(1, keepdim=True) / case["cols"] + EPS)
        if op == "norm":
            return {"y": y, "h": h}
        top = y.abs().max(dim=1).values
        scale = torch.where(top == 0, torch.ones_like(top), top / 448)
        return {"q": _e4m3(y / scale.unsqueeze(1)), "scale": scale, "h": h}
    if op == "norm_grad":
        h, w, dy = s["h"], s["weight"], s["dy"]
        ms = (h * h).sum(1, keepdim=True) / case["cols"] + EPS
        dot = (dy * w * h).sum(1, keepdim=True)
        return {"dx": s["dh"] + dy * w / ms.sqrt() - h * dot / (case["cols"] * ms ** 1.5), "dweight": (dy * h / ms.sqrt()).sum(0)}

    def act(v):
        if case["act"] == "silu":
            return v / (1 + torch.exp(-v))
        return v / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))

    def slope(v):
        if case["act"] == "silu":
            inner, up = v, torch.ones_like(v)
        else:
            inner = 2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)
            up = 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * v * v)
        p = 1 / (1 + torch.exp(-inner))
        return p + v * p * (1 - p) * up

    if op in ("ff", "ff8"):
        one = torch.ones((), dtype=torch.float64, device="cuda")
        x = s["x"] * s.get("x_scale", one).reshape(-1, 1)
        g = torch.mm(x, (s["w_gate"] * s.get("w_gate_scale", one).reshape(-1, 1)).t().contiguous())
        u = torch.mm(x, (s["w_up"] * s.get("w_up_scale", one).reshape(-1, 1)).t().contiguous())
        if case["bias"]:
            g += s["b_gate"]
            u += s["b_up"]
        h = u * act(g)
        return {"h": h, "gate": g, "up": u} if case.get("keep") else {"h": h}
    du = act(s["gate"]) * s["dh"]
    dg = slope(s["gate"]) * s["up"] * s["dh"]
    got = {"dx": torch.mm(dg, s["w_gate"]).add_(torch.mm(du, s["w_up"])),
           "dw_gate": torch.mm(dg.t().contiguous(), s["x"]), "dw_up": torch.mm(du.t().contiguous(), s["x"])}
    return dict(got, db_gate=dg.sum(0), db_up=du.sum(0)) if case["bias"] else got
