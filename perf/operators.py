"""The row-wise operators of this framework as cases that can be timed: each in its plain form, in elementary torch
operations, and as the calls of `anode_b200.ops` that a user makes.

Kinds
  norm         RMS norm with the residual's addition, forward: y, the sum, and for training each row's 1/rms
  norm_grad    its adjoint: dx (which is the residual's gradient, too) and dgamma
  quant        the same norm with its output in 8 bits (e4m3) and scales: one per row, or one per 128 columns
  rotary       rotary positions of queries and keys, with or without the RMS norm of each head before them
  rotary_grad  the adjoint: dq, dk and the gradients of the norms' weights

Formulas (rounded to the tensors' type once, at the end; the norm reads the sum as it is stored)
  t = round(x + residual),  r = (mean(t^2) + epsilon)^-1/2,  y = t*r*gamma
  g = dy*gamma, xh = t*r:   dx = r*(g - xh*mean(g*xh)) + dt,  dgamma = sum over rows of dy*xh
  a = max |y| of a group:   scale = max(a, 2^-96)/448,  q = e4m3(y/scale)
  angle = position*freq[i]: (u, v) -> A*(u cos - v sin, u sin + v cos), i below half the rotated width; the pairs
  are (i, i + half) or, interleaved, (2i, 2i + 1); the rest of the head passes unchanged

Ranges: 1 to 16384 rows of 32 to 16384 columns; 1 to 16384 tokens of 1 to 64 heads of 16 to 256 elements, all or part
of which are rotated, positions up to a million; f32, f16 and bf16.
"""
import math

import torch

own = False          # False: the plain forms; True: the framework's operators

EPSILON = 1e-5
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TINY, E4M3 = 2.0 ** -96, 448.0


def _rows(kind, type, rows, cols, **options):
    case = dict(kind=kind, type=type, rows=rows, cols=cols, residual=True, save=False, block=0)
    case.update(options)
    return case


def _heads(kind, type, tokens, heads, kv_heads, dim, rot, **options):
    case = dict(kind=kind, type=type, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rot=rot, interleaved=False, norm=False,
                stretch=1.0, start=0, packed=False)
    case.update(options)
    return case


def listed():
    return [
        # one new token through a layer's norm: nothing but latency
        _rows("norm", "bf16", 1, 4096, name="norm_token"),
        # a long prompt, or a training batch, of a wide model: the largest call
        _rows("norm", "bf16", 16384, 8192, save=True, name="norm_prompt"),
        # sizes that divide by nothing, without a residual: the first norm of a stack
        _rows("norm", "f32", 4099, 1001, residual=False, save=True, name="norm_ragged"),
        # the backward pass of an ordinary training batch
        _rows("norm_grad", "bf16", 8192, 4096, name="norm_grad"),
        # the backward pass over ragged rows
        _rows("norm_grad", "f16", 2047, 1535, name="norm_grad_ragged"),
        # a few tokens of a serving batch, on their way to an 8-bit product
        _rows("quant", "bf16", 16, 8192, block=128, name="quant_tokens"),
        # a prompt on its way to an 8-bit product, a scale per 128 columns
        _rows("quant", "bf16", 8192, 8192, block=128, name="quant_prompt"),
        # a scale per row, odd sizes
        _rows("quant", "f16", 3001, 2050, name="quant_rows"),
        # a serving batch's new tokens, far into a stretched context
        _heads("rotary", "bf16", 32, 32, 8, 128, 128, stretch=8.0, start=100000, packed=True, name="rotary_tokens"),
        # a prompt whose heads are normed first, read out of the packed projection
        _heads("rotary", "bf16", 16384, 32, 8, 128, 128, norm=True, packed=True, name="rotary_prompt"),
        # its backward pass at a training batch
        _heads("rotary_grad", "bf16", 8192, 32, 8, 128, 128, norm=True, name="rotary_grad"),
        # part of each head, interleaved pairs, odd counts of heads and tokens, without a norm
        _heads("rotary_grad", "f32", 1999, 7, 1, 80, 24, interleaved=True, name="rotary_grad_part"),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm_grad", "norm_grad", "quant", "quant", "rotary", "rotary", "rotary_grad", "rotary_grad"])
    type = rng.choice(["bf16", "bf16", "f16", "f32"])
    size = 4 if type == "f32" else 2
    if kind in ("norm", "norm_grad", "quant"):
        cols = _spread(rng, 32, 16384)
        if rng.random() < 0.6:
            cols = max(32, cols // 64 * 64)
        rows = _spread(rng, 1, min(16384, 250000000 // (size * cols)))
        case = _rows(kind, type, rows, cols, residual=rng.random() < 0.7)
        if kind == "norm":
            case["save"] = rng.random() < 0.5
        if kind == "quant":
            case["block"] = rng.choice([0, 128, 128])
        return case
    dim = rng.choice([16, 40, 64, 64, 80, 96, 128, 128, 128, 192, 256])
    rot = dim if rng.random() < 0.6 else max(2, int(dim * rng.uniform(0.2, 0.9)) // 2 * 2)
    kv_heads = rng.choice([1, 1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 7, 8])
    tokens = _spread(rng, 1, min(16384, 200000000 // (size * (heads + kv_heads) * dim)))
    return _heads(kind, type, tokens, heads, kv_heads, dim, rot, interleaved=rng.random() < 0.4, norm=rng.random() < 0.5,
                  stretch=rng.choice([1.0, 1.0, 4.0, 8.0]), start=rng.choice([0, 0, rng.randrange(1000000)]), packed=rng.random() < 0.5)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * seed + 17)
    type = TYPES[case["type"]]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device="cuda", dtype=type) * scale

    def weights(n):
        return (1.0 + 0.1 * torch.randn(n, generator=g, device="cuda")).to(type)

    s = dict(case)
    if case["kind"] in ("norm", "norm_grad", "quant"):
        rows, cols = case["rows"], case["cols"]
        # a residual stream: most columns of size one, one in 64 much larger
        wide = torch.where(torch.rand(cols, generator=g, device="cuda") < 1 / 64, 16.0, 1.0).to(type)
        s["gamma"] = weights(cols)
        if case["kind"] == "norm_grad":
            s["total"] = normal(rows, cols) * wide
            s["inv_rms"] = (s["total"].float().square().mean(1) + EPSILON).rsqrt()
            s["dy"] = normal(rows, cols)
            s["dtotal"] = normal(rows, cols) if case["residual"] else None
            s["dx"], s["dgamma"] = torch.empty_like(s["dy"]), torch.empty_like(s["gamma"])
            return s
        s["x"] = normal(rows, cols)
        s["residual"] = normal(rows, cols) * wide if case["residual"] else None
        s["total"] = torch.empty_like(s["x"]) if case["residual"] else None
        if case["kind"] == "norm":
            s["y"] = torch.empty_like(s["x"])
            s["inv_rms"] = torch.empty(rows, device="cuda") if case["save"] else None
        else:
            s["q"] = torch.empty(rows, cols, device="cuda", dtype=torch.float8_e4m3fn)
            s["scale"] = torch.empty((rows, -(-cols // case["block"])) if case["block"] else (rows,), device="cuda")
        return s
    tokens, heads, kv, dim, rot = (case[k] for k in ("tokens", "heads", "kv_heads", "dim", "rot"))
    # frequencies of a context stretched by a factor: the slow ones divided by it, the fast ones kept, a ramp between
    freq = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    turns = 8192 * freq / (2 * math.pi)
    keep = ((turns - 1) / 3).clamp(0, 1)
    s["freq"] = freq * (keep + (1 - keep) / case["stretch"])
    s["amplitude"] = 1.0 + 0.1 * math.log(case["stretch"])
    step = 1 if tokens > 64 else 977          # a prompt's positions in turn; new tokens' are their sequences' lengths
    s["positions"] = case["start"] + step * torch.arange(tokens, device="cuda")
    if case["packed"]:
        both = normal(tokens, heads + 2 * kv, dim)
        q, k = both[:, :heads], both[:, heads:heads + kv]
    else:
        q, k = normal(tokens, heads, dim), normal(tokens, kv, dim)
    s["q"], s["k"] = q, k
    s["gamma_q"], s["gamma_k"] = (weights(dim), weights(dim)) if case["norm"] else (None, None)
    s["epsilon"] = EPSILON if case["norm"] else None
    s["q_out"], s["k_out"] = (torch.empty(tokens, h, dim, device="cuda", dtype=type) for h in (heads, kv))
    if case["kind"] == "rotary_grad":
        s["dq"], s["dk"] = normal(tokens, heads, dim), normal(tokens, kv, dim)
        s["dgamma_q"], s["dgamma_k"] = (torch.empty_like(w) if w is not None else None for w in (s["gamma_q"], s["gamma_k"]))
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------------------

def _sum(s):
    return s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(s["x"].dtype)


def _norm(s):
    total = _sum(s)
    t = total.float()
    r = 1.0 / torch.sqrt((t * t).mean(1) + EPSILON)
    return total, r, t * r[:, None] * s["gamma"].float()


def _plain_norm(s):
    total, r, y = _norm(s)
    return {"y": y.to(total.dtype), "total": None if s["residual"] is None else total, "inv_rms": r if s["save"] else None}


def _plain_norm_grad(s):
    t, dy, r = s["total"].float(), s["dy"].float(), s["inv_rms"][:, None]
    g, xh = dy * s["gamma"].float(), t * r
    dx = r * (g - xh * (g * xh).mean(1, keepdim=True))
    if s["dtotal"] is not None:
        dx = dx + s["dtotal"].float()
    return {"dx": dx.to(s["dy"].dtype), "dgamma": (dy * xh).sum(0).to(s["gamma"].dtype)}


def _plain_quant(s):
    total, _, y = _norm(s)
    rows, cols = y.shape
    width = s["block"] or cols
    groups = -(-cols // width)
    y = torch.nn.functional.pad(y, (0, groups * width - cols)).view(rows, groups, width)
    scale = y.abs().amax(2).clamp(min=TINY) / E4M3
    q = (y / scale[:, :, None]).clamp(-E4M3, E4M3).view(rows, groups * width)[:, :cols].contiguous().to(torch.float8_e4m3fn)
    return {"q": q, "scale": scale if s["block"] else scale[:, 0], "total": None if s["residual"] is None else total}


def _cos_sin(s):
    angle = s["positions"].double()[:, None] * s["freq"]
    return (s["amplitude"] * torch.cos(angle)).float()[:, None], (s["amplitude"] * torch.sin(angle)).float()[:, None]


def _turn(s, x, cos, sin):
    rot, half = s["rot"], s["rot"] // 2
    if s["interleaved"]:
        u, v = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((u * cos - v * sin, u * sin + v * cos), -1).flatten(-2)
    else:
        u, v = x[..., :half], x[..., half:rot]
        turned = torch.cat((u * cos - v * sin, u * sin + v * cos), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _plain_rotary(s):
    cos, sin = _cos_sin(s)

    def one(x, gamma):
        n = x.float()
        if gamma is not None:
            n = n / torch.sqrt((n * n).mean(-1, keepdim=True) + EPSILON) * gamma.float()
        return _turn(s, n, cos, sin).to(x.dtype)

    return {"q": one(s["q"], s["gamma_q"]), "k": one(s["k"], s["gamma_k"])}


def _plain_rotary_grad(s):
    cos, sin = _cos_sin(s)

    def one(dout, x, gamma):
        dn = _turn(s, dout.float(), cos, -sin)
        if gamma is None:
            return dn.to(x.dtype), None
        x = x.float()
        r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPSILON)
        g, xh = dn * gamma.float(), x * r
        return (r * (g - xh * (g * xh).mean(-1, keepdim=True))).to(dout.dtype), (dn * xh).sum((0, 1)).to(gamma.dtype)

    dq, dgamma_q = one(s["dq"], s["q"], s["gamma_q"])
    dk, dgamma_k = one(s["dk"], s["k"], s["gamma_k"])
    return {"dq": dq, "dk": dk, "dgamma_q": dgamma_q, "dgamma_k": dgamma_k}


# ---- the framework's operators --------------------------------------------------------------------------------------------

def _own(s):
    from anode_b200 import ops
    kind = s["kind"]
    if kind == "norm":
        ops.RmsNormalizeAddOp.apply(EPSILON, s["x"], s["y"], s["gamma"], s["residual"], s["total"], s["inv_rms"])
        return {"y": s["y"], "total": s["total"], "inv_rms": s["inv_rms"]}
    if kind == "norm_grad":
        ops.RmsNormalizeAddOp.adjoint(s["dy"], s["total"], s["inv_rms"], s["dx"], s["gamma"], s["dtotal"], s["dgamma"])
        return {"dx": s["dx"], "dgamma": s["dgamma"]}
    if kind == "quant":
        ops.RmsNormalizeAddQuantOp.apply(EPSILON, s["x"], s["q"], s["scale"], s["gamma"], s["residual"], s["total"])
        return {"q": s["q"], "scale": s["scale"], "total": s["total"]}
    if kind == "rotary":
        ops.RotaryPositionsOp.apply(s["positions"], s["freq"], s["q"], s["k"], s["q_out"], s["k_out"], s["interleaved"], s["amplitude"],
                                    s["epsilon"], s["gamma_q"], s["gamma_k"])
        return {"q": s["q_out"], "k": s["k_out"]}
    ops.RotaryPositionsOp.adjoint(s["positions"], s["freq"], s["dq"], s["dk"], s["q_out"], s["k_out"], s["interleaved"], s["amplitude"],
                                  s["epsilon"], s["q"], s["k"], s["gamma_q"], s["gamma_k"], s["dgamma_q"], s["dgamma_k"])
    return {"dq": s["q_out"], "dk": s["k_out"], "dgamma_q": s["dgamma_q"], "dgamma_k": s["dgamma_k"]}


_PLAIN = {"norm": _plain_norm, "norm_grad": _plain_norm_grad, "quant": _plain_quant, "rotary": _plain_rotary, "rotary_grad": _plain_rotary_grad}


def run(state):
    return _own(state) if own else _PLAIN[state["kind"]](state)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------

def _e4m3_64(v):
    """The nearest e4m3 value of each |v| <= 448, ties to even: steps of 2^-3 of the leading power of two, no finer than 2^-9."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), e.clamp(min=-5) - 4)
    return torch.round(v / step) * step


def _complex(s, sign):
    angle = s["positions"].double().unsqueeze(1) * s["freq"].unsqueeze(0)
    return torch.polar(torch.full_like(angle, s["amplitude"]), sign * angle).unsqueeze(1)


def _turn_64(s, x, by):
    rot, half = s["rot"], s["rot"] // 2
    index = torch.arange(rot, device=x.device)
    first, second = (index[0::2], index[1::2]) if s["interleaved"] else (index[:half], index[half:])
    z = torch.complex(x[..., first], x[..., second]) * by
    out = x.clone()
    out[..., first], out[..., second] = z.real, z.imag
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("norm", "quant"):
        t = s["x"].double()
        if s["residual"] is not None:
            t = (t + s["residual"].double()).to(s["x"].dtype).double()
        mean_square = torch.linalg.vector_norm(t, dim=1).square() / case["cols"]
        r = (mean_square + EPSILON).pow(-0.5)
        y = torch.mul(t, r.unsqueeze(1)).mul_(s["gamma"].double())
        total = t if s["residual"] is not None else None
        if kind == "norm":
            return {"y": y, "total": total, "inv_rms": r if case["save"] else None}
        width = case["block"] or case["cols"]
        column = torch.arange(case["cols"], device=y.device) // width
        peak = torch.zeros(case["rows"], int(column[-1]) + 1, device=y.device, dtype=torch.float64)
        peak = peak.scatter_reduce(1, column.expand(case["rows"], -1), y.abs(), "amax")
        scale = torch.clamp(peak, min=TINY) / E4M3
        q = _e4m3_64(y / scale[:, column])
        return {"q": q, "scale": scale if case["block"] else scale.squeeze(1), "total": total}
    if kind == "norm_grad":
        # d/dt of gamma*t*r:  r*g - t*r^3*(g.t)/cols
        t, dy, r = s["total"].double(), s["dy"].double(), s["inv_rms"].double().unsqueeze(1)
        g = dy * s["gamma"].double()
        along = torch.linalg.vecdot(g, t).unsqueeze(1) / case["cols"]
        dx = g.mul_(r).sub_(t * r.pow(3) * along)
        if s["dtotal"] is not None:
            dx = dx.add_(s["dtotal"].double())
        return {"dx": dx, "dgamma": torch.einsum("rc,rc,r->c", dy, t, r.squeeze(1))}
    if kind == "rotary":
        by = _complex(s, 1.0)

        def forward(x, gamma):
            x = x.double()
            if gamma is not None:
                x = x * (x.square().mean(-1, keepdim=True) + EPSILON).pow(-0.5) * gamma.double()
            return _turn_64(s, x, by)

        return {"q": forward(s["q"], s["gamma_q"]), "k": forward(s["k"], s["gamma_k"])}
    by = _complex(s, -1.0)

    def backward(dout, x, gamma):
        dn = _turn_64(s, dout.double(), by)
        if gamma is None:
            return dn, None
        x = x.double()
        r = (x.square().mean(-1, keepdim=True) + EPSILON).pow(-0.5)
        g = dn * gamma.double()
        along = torch.linalg.vecdot(g, x).unsqueeze(-1) / case["dim"]
        return g * r - x * r.pow(3) * along, torch.einsum("thd,thd,th->d", dn, x, r.squeeze(-1))

    dq, dgamma_q = backward(s["dq"], s["q"], s["gamma_q"])
    dk, dgamma_k = backward(s["dk"], s["k"], s["gamma_k"])
    return {"dq": dq, "dk": dk, "dgamma_q": dgamma_q, "dgamma_k": dgamma_k}


def work(case):
    e = 4 if case["type"] == "f32" else 2
    kind = case["kind"]
    if kind in ("norm", "norm_grad", "quant"):
        rows, cols = case["rows"], case["cols"]
        n, more = rows * cols, 1 if case["residual"] else 0
        if kind == "norm":        # x, residual, gamma; y, total, inv_rms
            return {"bytes": n * e * (2 + 2 * more) + cols * e + (4 * rows if case["save"] else 0), "flops": n * (4 + more)}
        if kind == "norm_grad":   # dy, total, dtotal, inv_rms, gamma; dx, dgamma
            return {"bytes": n * e * (3 + more) + 4 * rows + 2 * cols * e, "flops": n * (10 + more)}
        groups = rows * (-(-cols // case["block"]) if case["block"] else 1)
        return {"bytes": n * (e * (1 + 2 * more) + 1) + cols * e + 4 * groups, "flops": n * (6 + more)}
    n = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
    turned = 3 * case["tokens"] * (case["heads"] + case["kv_heads"]) * case["rot"]
    small = 8 * case["tokens"] + 4 * case["rot"]
    weight = 2 * case["dim"] * e if case["norm"] else 0
    if kind == "rotary":
        return {"bytes": 2 * n * e + small + weight, "flops": turned + (4 * n if case["norm"] else 0)}
    return {"bytes": (3 if case["norm"] else 2) * n * e + small + 2 * weight, "flops": turned + (11 * n if case["norm"] else 0)}
