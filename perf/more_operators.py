"""The operators at the two ends of a language model and between its layers, as cases that can be timed: each in its plain form,
in elementary torch operations, and as the calls of `anode_b200.ops` that a user makes.

Kinds
  layer         layer norm with the residual's addition, forward: y, the sum, and for training each row's mean and 1/std
  layer_grad    its adjoint: dx (which is the residual's gradient, too), dgamma and dbeta
  embed         rows of a table by tokens, times a scale
  embed_grad    the table's gradient: the sum of the rows of each token, over the whole table; in a step of two micro-batches the
                second one adds to the first one's
  logprob       log probabilities of given tokens with their rows' entropies, and the likeliest tokens with theirs
  logprob_grad  the gradient of the logits from those of the log probabilities and the entropies

Formulas (rounded to the tensors' type once, at the end; the norm reads the sum as it is stored)
  t = round(x + residual),  mu = mean(t),  r = (mean((t - mu)^2) + epsilon)^-1/2,  y = (t - mu)*r*gamma + beta
  g = dy*gamma, xh = (t - mu)*r:   dx = r*(g - mean(g) - xh*mean(g*xh)) + dt,  dgamma = sum of dy*xh, dbeta = sum of dy over rows
  y[i] = scale*table[token[i]],  dtable[v] = scale * sum of dy[i] over token[i] = v;   a token outside of the table has a row of
  zeros and no gradient
  m = max x, z = scale*(x - m), L = log(sum(exp(z))):   logprob = z[token] - L,  H = L - sum(z*exp(z))/sum(exp(z)),  and the
  row keeps (m, L);  a token outside of the row has log probability 0 and no gradient; a row whose x are all -infinity has
  log probability -infinity, entropy 0, L = 0 and no gradient; the likeliest tokens come in falling order, ties by the lowest index
  p = exp(z - L):   dx = scale*(dlogprob*([token] - p) - dentropy*p*(z - L + H))

Ranges: layer norms of 1 to 16384 rows of 32 to 16384 columns; 1 to 32768 tokens out of tables of 16 to 262144 rows of 16 to 8192
columns; 1 to 8192 rows of 64 to 262144 logits, with up to 64 alternatives; f32, f16 and bf16.
"""
import math

import torch

own = False          # False: the plain forms; True: the framework's operators

EPSILON = 1e-5
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _rows(kind, type, rows, cols, **options):
    case = dict(kind=kind, type=type, rows=rows, cols=cols, residual=True, save=False)
    case.update(options)
    return case


def _table(kind, type, tokens, vocab, cols, **options):
    # holes: the share of tokens that stand for none; sums: the type of the table's gradient; steps: micro-batches that add up
    case = dict(kind=kind, type=type, tokens=tokens, vocab=vocab, cols=cols, scale=1.0, holes=0.0, sums=type, steps=1)
    case.update(options)
    return case


def _logits(kind, type, rows, vocab, **options):
    # kept: the share of a row's logits that a mask leaves; holes: the share of tokens that stand for none; entropy: asked for, too
    case = dict(kind=kind, type=type, rows=rows, vocab=vocab, scale=1.0, top=0, kept=1.0, holes=0.0, entropy=True, save=False)
    case.update(options)
    return case


def listed():
    return [
        # one new token through a layer's norm: nothing but latency
        _rows("layer", "bf16", 1, 4096, name="layer_token"),
        # a long prompt, or a training batch, of a wide model: the largest norm
        _rows("layer", "bf16", 16384, 8192, save=True, name="layer_prompt"),
        # sizes that divide by nothing, without a residual: the first norm of a stack
        _rows("layer", "f32", 4099, 1001, residual=False, save=True, name="layer_ragged"),
        # the backward pass of an ordinary training batch
        _rows("layer_grad", "bf16", 8192, 4096, name="layer_grad"),
        # the backward pass over ragged rows
        _rows("layer_grad", "f16", 2047, 1535, name="layer_grad_ragged"),
        # a serving batch's new tokens
        _table("embed", "bf16", 32, 131072, 4096, scale=64.0, name="embed_tokens"),
        # a long prompt, or a training batch, with padding
        _table("embed", "bf16", 16384, 32768, 8192, holes=0.05, name="embed_prompt"),
        # the backward pass of an ordinary training batch: the whole table's gradient
        _table("embed_grad", "bf16", 16384, 32768, 4096, scale=64.0, name="embed_grad"),
        # two micro-batches into gradients in 32 bits, ragged sizes
        _table("embed_grad", "f16", 4099, 50021, 1001, sums="f32", steps=2, holes=0.05, name="embed_grad_two"),
        # a serving batch: the chosen tokens' log probabilities and the likeliest twenty
        _logits("logprob", "f32", 16, 131072, scale=1.25, top=20, name="logprob_tokens"),
        # a training batch with a large vocabulary: the largest call
        _logits("logprob", "bf16", 4096, 131072, holes=0.1, save=True, name="logprob_batch"),
        # its backward pass, over rows that begin anywhere
        _logits("logprob_grad", "bf16", 4096, 50021, holes=0.1, name="logprob_grad"),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["layer", "layer_grad", "embed", "embed_grad", "logprob", "logprob_grad"])
    type = rng.choice(["bf16", "bf16", "f16", "f32"])
    size = 4 if type == "f32" else 2
    if kind in ("layer", "layer_grad"):
        cols = _spread(rng, 32, 16384)
        if rng.random() < 0.6:
            cols = max(32, cols // 64 * 64)
        rows = _spread(rng, 1, min(16384, 250000000 // (size * cols)))
        case = _rows(kind, type, rows, cols, residual=rng.random() < 0.7)
        if kind == "layer":
            case["save"] = rng.random() < 0.5
        return case
    if kind in ("embed", "embed_grad"):
        cols = _spread(rng, 16, 8192)
        if rng.random() < 0.6:
            cols = max(16, cols // 16 * 16)
        vocab = _spread(rng, 16, min(262144, 250000000 // (size * cols)))
        tokens = _spread(rng, 1, min(32768, 250000000 // (size * cols)))
        case = _table(kind, type, tokens, vocab, cols, scale=rng.choice([1.0, 1.0, 8.0, 45.25]), holes=rng.choice([0.0, 0.0, 0.1]))
        if kind == "embed_grad":
            case["sums"] = rng.choice([type, "f32"])
            case["steps"] = rng.choice([1, 1, 2])
        return case
    vocab = _spread(rng, 64, 262144)
    if rng.random() < 0.5:
        vocab = max(64, vocab // 64 * 64)
    rows = _spread(rng, 1, min(8192, 500000000 // (size * vocab)))
    case = _logits(kind, type, rows, vocab, scale=rng.choice([1.0, 1.0, 0.7, 2.0]), kept=rng.choice([1.0, 1.0, 0.2]), holes=rng.choice([0.0, 0.1]),
                   entropy=rng.random() < 0.6)
    if kind == "logprob":
        case["save"] = rng.random() < 0.5
        if rows * vocab <= 50000000:
            case["top"] = rng.choice([0, 1, 5, 20, 64])
    return case


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * seed + 17)
    type = TYPES[case["type"]]
    kind = case["kind"]

    def normal(*shape, dtype=type):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype)

    def uniform(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    def tokens_of(n, vocab, none):
        # the few common ones low and often, as a vocabulary ordered by frequency has them
        t = (torch.exp(uniform(n).double() * math.log(vocab + 1)).long() - 1).clamp(0, vocab - 1)
        return torch.where(uniform(n) < case["holes"], none, t)

    s = dict(case)
    if kind in ("layer", "layer_grad"):
        rows, cols = case["rows"], case["cols"]
        # a residual stream: most columns of size one, one in 64 much larger and away from zero
        far = uniform(cols) < 1 / 64
        wide, middle = torch.where(far, 16.0, 1.0).to(type), torch.where(far, 8.0, 0.25).to(type)
        s["gamma"] = (1.0 + 0.1 * normal(cols, dtype=torch.float32)).to(type)
        s["beta"] = (0.1 * normal(cols, dtype=torch.float32)).to(type)
        if kind == "layer_grad":
            s["total"] = normal(rows, cols) * wide + middle
            t = s["total"].double()
            s["mean"] = t.mean(1).float()
            s["inv_std"] = (t.var(1, correction=0) + EPSILON).rsqrt().float()
            s["dy"] = normal(rows, cols)
            s["dtotal"] = normal(rows, cols) if case["residual"] else None
            s["dx"], s["dgamma"], s["dbeta"] = torch.empty_like(s["dy"]), torch.empty_like(s["gamma"]), torch.empty_like(s["beta"])
            return s
        if case["residual"]:
            s["x"], s["residual"] = normal(rows, cols), normal(rows, cols) * wide + middle
            s["total"] = torch.empty_like(s["x"])
        else:
            s["x"], s["residual"], s["total"] = normal(rows, cols) * wide + middle, None, None
        s["y"] = torch.empty_like(s["x"])
        s["mean"], s["inv_std"] = (torch.empty(rows, device="cuda") if case["save"] else None for _ in range(2))
        return s
    if kind == "embed":
        s["table"] = normal(case["vocab"], case["cols"])
        s["token"] = tokens_of(case["tokens"], case["vocab"], -1)
        s["y"] = torch.empty(case["tokens"], case["cols"], device="cuda", dtype=type)
        return s
    if kind == "embed_grad":
        s["token"] = [tokens_of(case["tokens"], case["vocab"], -1) for _ in range(case["steps"])]
        s["dy"] = [normal(case["tokens"], case["cols"]) for _ in range(case["steps"])]
        s["dtable"] = torch.empty(case["vocab"], case["cols"], device="cuda", dtype=TYPES[case["sums"]])
        return s
    rows, vocab = case["rows"], case["vocab"]
    s["token"] = tokens_of(rows, vocab, -100)
    # logits as a model gives them: a spread of 3, the next token's well above it in most rows
    x = normal(rows, vocab).mul_(3.0)
    at = s["token"].clamp(min=0)[:, None]
    x.scatter_add_(1, at, (8.0 * uniform(rows, 1)).to(type))
    if case["kept"] < 1:
        x.masked_fill_((uniform(1, vocab) >= case["kept"]).expand(rows, -1).scatter(1, at, False), -math.inf)
    s["logits"] = x
    if kind == "logprob":
        s["logprob"] = torch.empty(rows, device="cuda")
        s["entropy_out"] = torch.empty(rows, device="cuda") if case["entropy"] else None
        s["stats"] = torch.empty(rows, 2, device="cuda") if case["save"] else None
        s["top_logprob"] = torch.empty(rows, case["top"], device="cuda") if case["top"] else None
        s["top_token"] = torch.empty(rows, case["top"], device="cuda", dtype=torch.int64) if case["top"] else None
        return s
    plain = _plain_logprob(dict(s, save=True, top=0, entropy=True))
    s["stats"], s["entropy_in"] = plain["stats"], plain["entropy"] if case["entropy"] else None
    s["dlogprob"] = normal(rows, dtype=torch.float32) / rows
    s["dentropy"] = normal(rows, dtype=torch.float32) / rows if case["entropy"] else None
    s["dlogits"] = torch.empty_like(x)
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------------------

def _plain_layer(s):
    x = s["x"].float()
    total = s["x"] if s["residual"] is None else (x + s["residual"].float()).to(s["x"].dtype)
    t = total.float()
    mean = t.mean(1)
    c = t - mean[:, None]
    r = 1.0 / torch.sqrt((c * c).mean(1) + EPSILON)
    y = (c * r[:, None] * s["gamma"].float() + s["beta"].float()).to(total.dtype)
    return {"y": y, "total": None if s["residual"] is None else total, "mean": mean if s["save"] else None, "inv_std": r if s["save"] else None}


def _plain_layer_grad(s):
    dy, r = s["dy"].float(), s["inv_std"][:, None]
    g, xh = dy * s["gamma"].float(), (s["total"].float() - s["mean"][:, None]) * r
    dx = r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    if s["dtotal"] is not None:
        dx = dx + s["dtotal"].float()
    return {"dx": dx.to(s["dy"].dtype), "dgamma": (dy * xh).sum(0).to(s["gamma"].dtype), "dbeta": dy.sum(0).to(s["beta"].dtype)}


def _plain_embed(s):
    inside = (s["token"] >= 0) & (s["token"] < s["vocab"])
    rows = s["table"][torch.where(inside, s["token"], 0)].float() * s["scale"]
    return {"y": torch.where(inside[:, None], rows, 0.0).to(s["table"].dtype)}


def _plain_embed_grad(s):
    def one(token, dy):
        inside = (token >= 0) & (token < s["vocab"])
        sums = torch.zeros(s["vocab"], s["cols"], device=dy.device)
        return sums.index_add_(0, torch.where(inside, token, 0), torch.where(inside[:, None], dy.float(), 0.0)) * s["scale"]

    out = one(s["token"][0], s["dy"][0]).to(s["dtable"].dtype)
    for token, dy in zip(s["token"][1:], s["dy"][1:]):
        out = (out.float() + one(token, dy)).to(out.dtype)
    return {"dtable": out}


def _shifted(s):
    """(m, z, empty): a row's largest logit, scale*(x - m), and whether the row has nothing but -infinity."""
    x = s["logits"].float()
    m = x.amax(1, keepdim=True)
    empty = m == -math.inf
    return m, (x - torch.where(empty, 0.0, m)) * s["scale"], empty


def _plain_logprob(s):
    m, z, empty = _shifted(s)
    e = torch.exp(z)
    total = torch.where(empty, 1.0, e.sum(1, keepdim=True))
    log_sum = torch.log(total)
    inside = (s["token"] >= 0) & (s["token"] < s["vocab"])
    picked = z.gather(1, torch.where(inside, s["token"], 0)[:, None]) - log_sum
    out = {"logprob": torch.where(inside, picked[:, 0], 0.0)}
    if s["entropy"]:
        out["entropy"] = torch.where(empty, 0.0, log_sum - torch.where(e > 0, e * z, 0.0).sum(1, keepdim=True) / total)[:, 0]
    if s["save"]:
        out["stats"] = torch.cat((m, log_sum), 1)
    if s["top"]:
        _, order = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True)
        out["top_token"] = order[:, :s["top"]].contiguous()
        out["top_logprob"] = z.gather(1, out["top_token"]) - log_sum
    return out


def _plain_logprob_grad(s):
    _, z, empty = _shifted(s)
    log_p = z - s["stats"][:, 1:]
    p = torch.exp(log_p)
    d = -p * s["dlogprob"][:, None]
    if s["dentropy"] is not None:
        d = d - torch.where(p > 0, s["dentropy"][:, None] * p * (log_p + s["entropy_in"][:, None]), 0.0)
    inside = ((s["token"] >= 0) & (s["token"] < s["vocab"]))[:, None]
    if s["holes"]:       # a token that stands for none takes its log probability's part away
        d = torch.where(inside, d, d + p * s["dlogprob"][:, None])
    d.scatter_add_(1, torch.where(inside, s["token"][:, None], 0), torch.where(inside, s["dlogprob"][:, None], 0.0))
    return {"dlogits": torch.where(empty, 0.0, d * s["scale"]).to(s["logits"].dtype)}


# ---- the framework's operators --------------------------------------------------------------------------------------------

def _own(s):
    from anode_b200 import ops
    kind = s["kind"]
    if kind == "layer":
        ops.LayerNormalizeAddOp.apply(EPSILON, s["x"], s["y"], s["gamma"], s["beta"], s["residual"], s["total"], s["mean"], s["inv_std"])
        return {"y": s["y"], "total": s["total"], "mean": s["mean"], "inv_std": s["inv_std"]}
    if kind == "layer_grad":
        ops.LayerNormalizeAddOp.adjoint(s["dy"], s["total"], s["mean"], s["inv_std"], s["dx"], s["gamma"], s["dtotal"], s["dgamma"], s["dbeta"])
        return {"dx": s["dx"], "dgamma": s["dgamma"], "dbeta": s["dbeta"]}
    if kind == "embed":
        ops.EmbedTokensOp.apply(s["token"], s["table"], s["y"], s["scale"])
        return {"y": s["y"]}
    if kind == "embed_grad":
        for i, (token, dy) in enumerate(zip(s["token"], s["dy"])):
            ops.EmbedTokensOp.adjoint(token, dy, s["dtable"], s["scale"], cap=ops.WriteCap.Accumulate if i else ops.WriteCap.Assign)
        return {"dtable": s["dtable"]}
    if kind == "logprob":
        ops.TokenLogProbsOp.apply(s["logits"], s["token"], s["logprob"], s["entropy_out"], s["stats"], s["top_logprob"], s["top_token"], s["scale"])
        names = {"logprob": "logprob", "entropy": "entropy_out", "stats": "stats", "top_token": "top_token", "top_logprob": "top_logprob"}
        return {name: s[at] for name, at in names.items() if s[at] is not None}
    ops.TokenLogProbsOp.adjoint(s["logits"], s["token"], s["stats"], s["dlogprob"], s["dlogits"], s["entropy_in"], s["dentropy"], s["scale"])
    return {"dlogits": s["dlogits"]}


_PLAIN = {"layer": _plain_layer, "layer_grad": _plain_layer_grad, "embed": _plain_embed, "embed_grad": _plain_embed_grad,
          "logprob": _plain_logprob, "logprob_grad": _plain_logprob_grad}


def run(state):
    return _own(state) if own else _PLAIN[state["kind"]](state)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------

def _exact_layer(s):
    t = s["x"].double()
    if s["residual"] is not None:
        t = torch.add(t, s["residual"].double()).to(s["x"].dtype).double()
    var, mean = torch.var_mean(t, dim=1, correction=0)
    r = torch.pow(var + EPSILON, -0.5)
    y = t.sub(mean.unsqueeze(1)).mul_(r.unsqueeze(1)).mul_(s["gamma"].double()).add_(s["beta"].double())
    return {"y": y, "total": t if s["residual"] is not None else None, "mean": mean if s["save"] else None, "inv_std": r if s["save"] else None}


def _exact_layer_grad(s):
    # the projection of r*g away from the ones and from t - mean
    dy, r = s["dy"].double(), s["inv_std"].double().unsqueeze(1)
    apart = s["total"].double().sub_(s["mean"].double().unsqueeze(1))
    g = torch.mul(dy, s["gamma"].double())
    along = torch.linalg.vecdot(g, apart).unsqueeze(1) / s["cols"]
    dgamma = torch.einsum("rc,rc,r->c", dy, apart, r.squeeze(1))
    dx = g.sub_(g.sum(1, keepdim=True) / s["cols"]).mul_(r).sub_(apart.mul_(along * r.pow(3)))
    return {"dx": dx if s["dtotal"] is None else dx.add_(s["dtotal"].double()), "dgamma": dgamma, "dbeta": dy.sum(0)}


def _exact_embed(s):
    known = s["token"].ge(0).logical_and(s["token"].lt(s["vocab"])).nonzero().squeeze(1)
    y = torch.zeros(s["tokens"], s["cols"], device="cuda", dtype=torch.float64)
    y[known] = s["table"].index_select(0, s["token"][known]).double().mul_(s["scale"])
    return {"y": y}


def _exact_embed_grad(s):
    # of the tokens in order: the differences of running sums where each one's run ends
    out = torch.zeros(s["vocab"], s["cols"], device="cuda", dtype=torch.float64)
    for token, dy in zip(s["token"], s["dy"]):
        order = torch.argsort(token)
        order = order[(token[order] >= 0) & (token[order] < s["vocab"])]
        which, count = torch.unique_consecutive(token[order], return_counts=True)
        if not which.numel():
            continue
        last = count.cumsum(0) - 1
        sums = dy[order].double().cumsum_(0)[last]
        sums[1:] -= sums[:-1].clone()
        step = sums.mul_(s["scale"])
        out[which] += step
        if s["steps"] > 1 and s["sums"] != "f32":
            out = out.to(s["dtable"].dtype).double()       # each step's sum as it is stored
    return {"dtable": out}


def _exact_logprob(s):
    parts = []
    for first in range(0, s["rows"], 512):
        x, token = s["logits"][first:first + 512].double(), s["token"][first:first + 512]
        z = x * s["scale"]
        whole = torch.logsumexp(z, 1)
        empty = whole.isinf()
        logs = z.sub_(whole.masked_fill(empty, 0.0).unsqueeze(1))
        known = token.ge(0).logical_and(token.lt(s["vocab"]))
        picked = torch.take_along_dim(logs, token.clamp(0, s["vocab"] - 1).unsqueeze(1), 1).squeeze(1)
        out = {"logprob": torch.where(known, picked, torch.zeros_like(picked))}
        if s["entropy"]:
            out["entropy"] = torch.special.entr(logs.exp()).sum(1)
        if s["save"]:
            m = x.max(1).values
            out["stats"] = torch.stack((m, torch.where(empty, torch.zeros_like(whole), whole - s["scale"] * m)), 1)
        if s["top"]:
            order = torch.argsort(-x, dim=1, stable=True)[:, :s["top"]]
            out["top_token"], out["top_logprob"] = order, torch.take_along_dim(logs, order, 1)
        parts.append(out)
    return {name: torch.cat([part[name] for part in parts]) for name in parts[0]}


def _exact_logprob_grad(s):
    parts = []
    for first in range(0, s["rows"], 512):
        part = slice(first, first + 512)
        x, token, kept = s["logits"][part].double(), s["token"][part], s["stats"][part].double()
        empty = x.max(1, keepdim=True).values.isinf()
        logs = (x * s["scale"]).sub_((s["scale"] * kept[:, :1] + kept[:, 1:]).masked_fill(empty, 0.0))
        p = logs.exp()
        known = token.ge(0).logical_and(token.lt(s["vocab"]))
        weight = (s["dlogprob"][part].double() * known).unsqueeze(1)
        d = p.neg().mul_(weight)
        if s["dentropy"] is not None:
            # p*log p and p of the entropy's gradient, without 0 * infinity
            d += s["dentropy"][part].double().unsqueeze(1) * (torch.special.entr(p) - p * s["entropy_in"][part].double().unsqueeze(1))
        row = known.nonzero().squeeze(1)
        d[row, token[row]] += weight.squeeze(1)[row]
        parts.append(d.mul_(s["scale"]).masked_fill_(empty, 0.0))
    return {"dlogits": torch.cat(parts)}


_EXACT = {"layer": _exact_layer, "layer_grad": _exact_layer_grad, "embed": _exact_embed, "embed_grad": _exact_embed_grad,
          "logprob": _exact_logprob, "logprob_grad": _exact_logprob_grad}


def exact(case, seed):
    return _EXACT[case["kind"]](prepare(case, seed))


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------

def _distinct(case):
    """The rows of the table that the tokens are expected to name."""
    at = torch.arange(case["vocab"], dtype=torch.float64)
    share = (1.0 - case["holes"]) * torch.log((at + 2) / (at + 1)) / math.log(case["vocab"] + 1)
    return int((1.0 - (1.0 - share) ** case["tokens"]).sum())


def work(case):
    e = 4 if case["type"] == "f32" else 2
    kind = case["kind"]
    if kind in ("layer", "layer_grad"):
        rows, cols = case["rows"], case["cols"]
        n, more = rows * cols, 1 if case["residual"] else 0
        if kind == "layer":       # x, residual, gamma, beta; y, total, mean, inv_std
            return {"bytes": n * e * (2 + 2 * more) + 2 * cols * e + (8 * rows if case["save"] else 0), "flops": n * (7 + more)}
        return {"bytes": n * e * (3 + more) + 8 * rows + 3 * cols * e, "flops": n * (13 + more)}      # dy, total, dtotal, mean, inv_std, gamma; dx, dgamma, dbeta
    if kind == "embed":           # the tokens, the rows that they name; y
        return {"bytes": 8 * case["tokens"] + (_distinct(case) + case["tokens"]) * case["cols"] * e, "flops": case["tokens"] * case["cols"]}
    if kind == "embed_grad":      # the tokens and dy; the table's gradient, and in later steps its rows that the tokens name, read and written
        step = case["tokens"] * (8 + case["cols"] * e)
        more = (case["steps"] - 1) * _distinct(case) * 2
        return {"bytes": case["steps"] * step + (case["vocab"] + more) * case["cols"] * (4 if case["sums"] == "f32" else 2),
                "flops": case["steps"] * case["tokens"] * case["cols"] * 2}
    n = case["rows"] * case["vocab"]
    if kind == "logprob":         # the logits and tokens; a few numbers of each row
        return {"bytes": n * e + case["rows"] * (8 + 4 + (4 if case["entropy"] else 0) + (8 if case["save"] else 0) + 12 * case["top"]),
                "flops": n * (6 if case["entropy"] else 4)}
    return {"bytes": 2 * n * e + case["rows"] * (8 + 8 + 4 + (8 if case["entropy"] else 0)), "flops": n * (8 if case["entropy"] else 5)}
