"""The operators between a network's encodings and its layers - layer norm, embedding lookup, routing to experts, products
grouped by expert - as measurable cases: what a program holds before the call (`prepare`), one pass through the public
entry points (`run` with `own`) or through elementary torch operations in 32 bits (`run` without), the work a pass cannot
do without (`work`) and its result in 64 bits (`exact`).

Kinds of cases (direction "forward": the result; "train": the result and the gradients of all that can have one)
  norm      qmlp.layer_norm over the rows of a feature matrix, parameters in float32
  embed     qmlp.embedding: rows of a table of latent codes, times a scale; a token outside the table is masked
  route     qmlp.route: the k best of every row's experts, their weights, and the order of the slots by expert
  exchange  qmlp.dispatch of feature rows to their experts' order, and qmlp.combine of such rows back, weighted
  experts   qmlp.expert_linear: one matrix product per expert over its run of rows
"""
import math
import os
import sys
from types import SimpleNamespace

import torch

own = False

DTYPES = {"float": torch.float32, "half": torch.float16, "bfloat16": torch.bfloat16}
BYTES = {"float": 4, "half": 2, "bfloat16": 2}
EPS = 1e-5


def _qmlp():
    path = os.path.abspath("quick-mlp_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import qmlp
    return qmlp


def listed():
    return [
        # one latent code normalised in front of an interactive query, where only latency counts
        dict(name="norm_forward_1x512", kind="norm", direction="forward", dtype="half", rows=1, channels=512),
        # the encoded features of a batch of points, as wide as the layers behind them, one point more than a power of two
        dict(name="norm_train_64kx64", kind="norm", direction="train", dtype="half", rows=65537, channels=64),
        # the activations of a wide model over a large batch
        dict(name="norm_train_32kx4096", kind="norm", direction="train", dtype="bfloat16", rows=32768, channels=4096),
        # codes of a frame's points during rendering, from a half table
        dict(name="embed_forward_256kx128", kind="embed", direction="forward", dtype="half", tokens=262147, rows=20000, channels=128,
             skew=0.0, masked=0.0, scale=1.0),
        # a code per image of a capture, a million points per step: every row is hit a thousand times
        dict(name="embed_train_1mx32", kind="embed", direction="train", dtype="float", tokens=1000003, rows=1000, channels=32,
             skew=0.0, masked=0.05, scale=1.0),
        # a vocabulary whose tokens follow a power law, some rows hot and many without a token
        dict(name="embed_train_64kx512", kind="embed", direction="train", dtype="float", tokens=65536, rows=50000, channels=512,
             skew=1.0, masked=0.0, scale=22.627417),
        # one query served: the smallest call of a router
        dict(name="route_forward_1x64", kind="route", direction="forward", dtype="half", tokens=1, experts=64, k=2, normalize=True,
             masked=0.0),
        # a training batch's router with its gradient, some experts switched off for some rows
        dict(name="route_train_256kx64", kind="route", direction="train", dtype="half", tokens=262147, experts=64, k=2, normalize=True,
             masked=0.1),
        # the feature rows of a training batch on their way to the experts and back, with all gradients
        dict(name="exchange_train_128kx256", kind="exchange", direction="train", dtype="half", tokens=131072, channels=256, experts=64, k=2),
        # one query served: two experts of 64, weights read once
        dict(name="experts_forward_2", kind="experts", direction="forward", dtype="half", rows=2, experts=64, n_in=1024, n_out=2048,
             bias=True, spread=0.5),
        # many small experts, each in charge of a part of the scene, a million points over them
        dict(name="experts_train_1mx64x64", kind="experts", direction="train", dtype="half", rows=1000003, experts=512, n_in=64, n_out=64,
             bias=True, spread=0.3),
        # a wide expert layer of a training step
        dict(name="experts_train_128kx1024", kind="experts", direction="train", dtype="bfloat16", rows=131072, experts=16, n_in=1024,
             n_out=1024, bias=True, spread=0.3),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _size(rng, low, high, step):
    """spread over the logarithm; more than half are multiples of `step`, the rest whatever comes, odd ones among them"""
    n = _log(rng, low, high)
    return max(low, n // step * step) if rng.random() < 0.6 else n


def draw(rng):
    kind = rng.choice(["norm", "norm", "embed", "embed", "route", "exchange", "experts", "experts", "experts"])
    c = dict(kind=kind, direction=rng.choice(["forward", "train", "train"]))
    if kind == "norm":
        c["dtype"] = rng.choice(["half", "bfloat16", "float"])
        c["channels"] = _size(rng, 5, 16384, 8)     # (below, the input's gradient is rounding alone)
        c["rows"] = _log(rng, 1, max(1, min(1 << 17, (1 << 26) // c["channels"])))
    elif kind == "embed":
        c["dtype"] = rng.choice(["half", "bfloat16", "float"])
        c["channels"] = _size(rng, 1, 1024, 8)
        c["tokens"] = _log(rng, 1, min(1 << 20, (1 << 26) // c["channels"]))
        c["rows"] = _log(rng, 1, min(1 << 18, (1 << 26) // c["channels"]))
        c["skew"] = rng.choice([0.0, 0.5, 1.0])
        c["masked"] = rng.choice([0.0, 0.0, 0.2])
        c["scale"] = rng.choice([1.0, math.sqrt(c["channels"])])
    elif kind == "route":
        c["dtype"] = rng.choice(["half", "bfloat16", "float"])
        c["experts"] = rng.choice([2, 4, 8, 16, 37, 64, 100, 128, 256])
        c["tokens"] = _log(rng, 1, min(1 << 18, (1 << 25) // c["experts"]))
        c["k"] = rng.randint(1, min(8, c["experts"]))
        c["normalize"] = rng.random() < 0.5
        c["masked"] = rng.choice([0.0, 0.1, 0.6])
    elif kind == "exchange":
        c["dtype"] = rng.choice(["half", "bfloat16", "float"])
        c["experts"] = rng.choice([2, 8, 64, 256])
        c["channels"] = _size(rng, 1, 4096, 8)
        c["k"] = rng.randint(1, min(8, c["experts"]))
        c["tokens"] = _log(rng, 1, max(1, min(1 << 17, (1 << 25) // (c["channels"] * c["k"]))))
    else:
        c["dtype"] = rng.choice(["half", "bfloat16"])
        c["experts"] = _log(rng, 1, 512)
        c["n_in"] = _size(rng, 8, 2048, 8)
        c["n_out"] = _size(rng, 8, min(2048, (1 << 25) // (c["n_in"] * c["experts"])) if c["n_in"] * c["experts"] < 1 << 21 else 16, 8)
        c["rows"] = _log(rng, 1, max(1, min(1 << 20, (1 << 35) // (c["n_in"] * c["n_out"]), (1 << 26) // (c["n_in"] + c["n_out"]))))
        c["bias"] = rng.random() < 0.7
        c["spread"] = rng.choice([0.0, 0.3, 0.6])
    return c


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _normal(gen, shape, dtype, std=1.0, mean=0.0):
    return (torch.randn(shape, device="cuda", generator=gen) * std + mean).to(DTYPES[dtype])


def _mask(gen, shape, share):
    return torch.rand(shape, device="cuda", generator=gen) < share


def _ranks(u, n, skew):
    """uniform numbers -> ranks in [0, n) whose density falls as (10 + rank) ** -skew"""
    low, high = 10.0, 10.0 + n
    if skew == 1.0:
        r = low * torch.exp(u * math.log(high / low))
    else:
        r = (low ** (1 - skew) + u * (high ** (1 - skew) - low ** (1 - skew))) ** (1 / (1 - skew))
    return (r - low).long().clamp_(0, n - 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c, s = case, SimpleNamespace(case=case)
    if c["kind"] == "norm":
        shape = (c["rows"], c["channels"])
        s.x = _normal(gen, shape, c["dtype"], 1.5, 0.3)
        s.weight = _normal(gen, (c["channels"],), "float", 0.1, 1.0)
        s.bias = _normal(gen, (c["channels"],), "float", 0.1)
        s.grad = _normal(gen, shape, c["dtype"]) if c["direction"] == "train" else None
    elif c["kind"] == "embed":
        # popularity falls with a power of the rank; which row has which rank is random
        ranks = _ranks(torch.rand(c["tokens"], device="cuda", generator=gen, dtype=torch.float64), c["rows"], c["skew"])
        s.tokens = torch.randperm(c["rows"], device="cuda", generator=gen)[ranks]
        if c["masked"] > 0:
            s.tokens[_mask(gen, (c["tokens"],), c["masked"])] = -1
        s.table = _normal(gen, (c["rows"], c["channels"]), c["dtype"], 0.5)
        s.grad = _normal(gen, (c["tokens"], c["channels"]), c["dtype"]) if c["direction"] == "train" else None
    elif c["kind"] == "route":
        s.logits = _normal(gen, (c["tokens"], c["experts"]), c["dtype"], 1.5)
        if c["masked"] > 0:
            s.logits[_mask(gen, s.logits.shape, c["masked"])] = -math.inf
        s.grad = _normal(gen, (c["tokens"], c["k"]), "float") if c["direction"] == "train" else None
    elif c["kind"] == "exchange":
        n, k, e = c["tokens"], c["k"], c["experts"]
        experts = torch.rand((n, e), device="cuda", generator=gen).argsort(dim=1)[:, :k].int()
        s.experts = experts.contiguous()
        order = torch.argsort(experts.reshape(-1), stable=True).int()
        s.positions = torch.empty_like(order)
        s.positions[order.long()] = torch.arange(n * k, device="cuda", dtype=torch.int32)
        s.positions = s.positions.reshape(n, k)
        s.order = order
        s.offsets = torch.nn.functional.pad(torch.bincount(experts.reshape(-1).long(), minlength=e).cumsum(0).int(), (1, 0))
        s.weights = torch.softmax(_normal(gen, (n, k), "float"), dim=1)
        s.x = _normal(gen, (n, c["channels"]), c["dtype"])
        s.y = _normal(gen, (n * k, c["channels"]), c["dtype"])
        train = c["direction"] == "train"
        s.grad_rows = _normal(gen, (n * k, c["channels"]), c["dtype"]) if train else None
        s.grad = _normal(gen, (n, c["channels"]), c["dtype"]) if train else None
    else:
        popular = torch.exp(torch.randn(c["experts"], device="cuda", generator=gen) * c["spread"]).double().cpu()
        bounds = torch.round(c["rows"] * popular.cumsum(0) / popular.sum()).int()
        s.offsets = torch.nn.functional.pad(bounds, (1, 0)).cuda()
        s.most = int(torch.diff(bounds, prepend=bounds.new_zeros(1)).max())      # the plan of a program that pads to the longest run
        s.x = _normal(gen, (c["rows"], c["n_in"]), c["dtype"])
        s.weight = _normal(gen, (c["experts"], c["n_out"], c["n_in"]), c["dtype"], c["n_in"] ** -0.5)
        s.bias = _normal(gen, (c["experts"], c["n_out"]), c["dtype"], 0.1) if c["bias"] else None
        s.grad = _normal(gen, (c["rows"], c["n_out"]), c["dtype"]) if c["direction"] == "train" else None
    if c["direction"] == "train":
        for name in ("x", "y", "weight", "bias", "table", "logits", "weights"):
            t = getattr(s, name, None)
            if t is not None:
                t.requires_grad_()
    return s


# ---- one pass through the framework ----------------------------------------------------------------------------------
def _own_pass(s):
    qmlp, c = _qmlp(), s.case
    train = c["direction"] == "train"
    if c["kind"] == "norm":
        y = qmlp.layer_norm(s.x, s.weight, s.bias, EPS)
        return [y.detach(), *torch.autograd.grad(y, [s.x, s.weight, s.bias], s.grad)] if train else [y]
    if c["kind"] == "embed":
        y = qmlp.embedding(s.tokens, s.table, c["scale"])
        return [y.detach(), *torch.autograd.grad(y, [s.table], s.grad)] if train else [y]
    if c["kind"] == "route":
        r = qmlp.route(s.logits, c["k"], c["normalize"])
        out = [r.weights.detach(), r.experts, r.order, r.positions, r.offsets]
        return out + list(torch.autograd.grad(r.weights, [s.logits], s.grad)) if train else out
    if c["kind"] == "exchange":
        r = qmlp.Routing(s.weights, s.experts, s.order, s.positions, s.offsets)
        rows, y = qmlp.dispatch(s.x, r), qmlp.combine(s.y, r)
        if not train:
            return [rows, y]
        return [rows.detach(), y.detach(), *torch.autograd.grad([rows, y], [s.x, s.y, s.weights], [s.grad_rows, s.grad])]
    y = qmlp.expert_linear(s.x, s.weight, s.offsets, s.bias)
    if not train:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, [s.x, s.weight] + ([s.bias] if c["bias"] else []), s.grad)]


# ---- the plain forms: elementary operations in 32 bits, rounded once at the end ----------------------------------------
def _plain_norm(s, c, dtype):
    x = s.x.float()
    centred = x - x.mean(dim=1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(dim=1, keepdim=True) + EPS)
    unit = centred * rstd
    out = [(unit * s.weight + s.bias).to(dtype)]
    if c["direction"] == "train":
        g = s.grad.float()
        gw = g * s.weight
        dx = rstd * (gw - gw.mean(dim=1, keepdim=True) - unit * (gw * unit).mean(dim=1, keepdim=True))
        out += [dx.to(dtype), (g * unit).sum(dim=0), g.sum(dim=0)]
    return out


def _plain_embed(s, c, dtype):
    inside = (s.tokens >= 0) & (s.tokens < c["rows"])
    rows = torch.where(inside, s.tokens, 0)
    out = [(s.table[rows].float() * c["scale"] * inside[:, None]).to(dtype)]
    if c["direction"] == "train":
        total = torch.zeros((c["rows"] + 1, c["channels"]), device="cuda")
        total.index_add_(0, torch.where(inside, s.tokens, c["rows"]), s.grad.float())
        out.append((total[:-1] * c["scale"]).to(dtype))
    return out


def _plain_route(s, c, dtype):
    z, k, n, e = s.logits.float(), c["k"], c["tokens"], c["experts"]
    best, at = torch.sort(z, dim=1, descending=True, stable=True)
    best, at = best[:, :k], at[:, :k]
    chosen = best > -math.inf
    top = torch.where(chosen[:, :1], best[:, :1], 0.0)
    share = torch.exp(best - top)
    total = share.sum(dim=1, keepdim=True) if c["normalize"] else torch.exp(z - top).sum(dim=1, keepdim=True)
    weights = torch.where(chosen, share / total, 0.0)
    experts = torch.where(chosen, at, -1).int()
    slots = torch.where(chosen, at, e).reshape(-1)
    order = torch.argsort(slots, stable=True)
    positions = torch.empty_like(order)
    positions[order] = torch.arange(n * k, device="cuda")
    counts = torch.bincount(slots, minlength=e + 1)[:e].cumsum(0)
    used = chosen.reshape(-1)
    out = [weights, experts, torch.where(used[order], order, -1).int(), torch.where(chosen, positions.reshape(n, k), -1).int(),
           torch.cat([counts.new_zeros(1), counts]).int()]
    if c["direction"] == "train":
        g = torch.where(chosen, s.grad, 0.0)
        mean = (g * weights).sum(dim=1, keepdim=True)
        if c["normalize"]:
            grad = torch.zeros_like(z).scatter_add_(1, at, weights * (g - mean))
        else:
            p = torch.where(z > -math.inf, torch.exp(z - top) / total, 0.0)
            grad = p * (torch.zeros_like(z).scatter_add_(1, at, g) - mean)
        out.append(grad.to(dtype))
    return out


def _plain_exchange(s, c, dtype):
    n, k = c["tokens"], c["k"]
    token, at = s.order.long() // k, s.positions.long()
    y = s.y.float()[at]
    out = [s.x[token], (s.weights[:, :, None] * y).sum(dim=1).to(dtype)]
    if c["direction"] == "train":
        g = s.grad.float()
        out.append(s.grad_rows.float()[at].sum(dim=1).to(dtype))
        out.append((s.weights.reshape(-1)[s.order.long()][:, None] * g[token]).to(dtype))
        out.append((g[:, None, :] * y).sum(dim=2))
    return out


def _plain_experts(s, c, dtype):
    rows = torch.arange(c["rows"], device="cuda")
    expert = torch.searchsorted(s.offsets[1:].long(), rows, right=True)
    x, w = s.x.float(), s.weight
    if c["rows"] <= 64 and c["direction"] == "forward":     # few rows: each with its expert's matrix
        y = torch.einsum("rk,rnk->rn", x, w[expert].float())
        return [(y + s.bias[expert].float() if c["bias"] else y).to(dtype)]
    slot = rows - s.offsets.long()[expert]
    w = w.float()
    padded = x.new_zeros((c["experts"], s.most, c["n_in"]))
    padded[expert, slot] = x
    y = torch.bmm(padded, w.transpose(1, 2))[expert, slot]
    out = [(y + s.bias.float()[expert] if c["bias"] else y).to(dtype)]
    if c["direction"] == "train":
        g = x.new_zeros((c["experts"], s.most, c["n_out"]))
        g[expert, slot] = s.grad.float()
        out += [torch.bmm(g, w)[expert, slot].to(dtype), torch.bmm(g.transpose(1, 2), padded).to(dtype)]
        if c["bias"]:
            out.append(g.sum(dim=1).to(dtype))
    return out


PLAIN = {"norm": _plain_norm, "embed": _plain_embed, "route": _plain_route, "exchange": _plain_exchange, "experts": _plain_experts}


def run(state):
    if own:
        return _own_pass(state)
    with torch.no_grad():   # the plain forms write their gradients out
        return PLAIN[state.case["kind"]](state, state.case, DTYPES[state.case["dtype"]])


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    c, train = case, case["direction"] == "train"
    b = BYTES[c["dtype"]]
    if c["kind"] == "norm":
        n = c["rows"] * c["channels"]
        # x in, y out; x was just read, so the gradient adds its own input and result
        return {"bytes": n * b * (4 if train else 2) + c["channels"] * 4 * (4 if train else 2), "flops": n * (22 if train else 8)}
    if c["kind"] == "embed":
        n, table = c["tokens"] * c["channels"], c["rows"] * c["channels"]
        total = c["tokens"] * 8 + min(n, table) * b + n * b
        return {"bytes": total + (n + table) * b if train else total, "flops": n * (2 if train else 1)}
    if c["kind"] == "route":
        n, slots = c["tokens"] * c["experts"], c["tokens"] * c["k"]
        return {"bytes": n * b * (2 if train else 1) + slots * (20 if train else 16) + c["experts"] * 4, "flops": n * (8 if train else 4)}
    if c["kind"] == "exchange":
        n, slots = c["tokens"] * c["channels"], c["tokens"] * c["k"]
        rows = slots * c["channels"]
        forward = (2 * n + 2 * rows) * b + slots * 12
        return {"bytes": forward + (2 * n + 2 * rows) * b + slots * 4 if train else forward, "flops": rows * (7 if train else 2)}
    matrices = min(c["experts"], c["rows"]) * c["n_in"] * c["n_out"]
    flops = 2 * c["rows"] * c["n_in"] * c["n_out"]
    forward = (c["rows"] * (c["n_in"] + c["n_out"]) + matrices) * b
    if not train:
        return {"bytes": forward, "flops": flops}
    return {"bytes": forward + (c["rows"] * (c["n_in"] + c["n_out"]) + c["experts"] * c["n_in"] * c["n_out"]) * b, "flops": 3 * flops}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
@torch.no_grad()
def exact(case, seed):
    s, c, train = prepare(case, seed), case, case["direction"] == "train"
    f64 = torch.float64
    if c["kind"] == "norm":
        x, w, b = s.x.to(f64), s.weight.to(f64), s.bias.to(f64)
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        sigma = (var + EPS).sqrt()
        y = (x - mean) / sigma * w + b
        if not train:
            return [y]
        g = s.grad.to(f64)
        # the derivative of (x_j - mean) / sigma by x_i, contracted with g * w
        d = g * w
        dot = (d * (x - mean)).sum(dim=1, keepdim=True)
        dx = d / sigma - d.sum(dim=1, keepdim=True) / (c["channels"] * sigma) - (x - mean) * dot / (c["channels"] * sigma ** 3)
        return [y, dx, ((x - mean) / sigma * g).sum(dim=0), g.sum(dim=0)]
    if c["kind"] == "embed":
        table = torch.cat([s.table.to(f64), torch.zeros((1, c["channels"]), device="cuda", dtype=f64)])
        token = torch.where(s.tokens < 0, c["rows"], s.tokens)
        y = table.index_select(0, token) * c["scale"]
        if not train:
            return [y]
        total = torch.zeros_like(table)
        order = token.argsort()
        total.index_add_(0, token[order], s.grad.to(f64)[order] * c["scale"])
        return [y, total[:-1]]
    if c["kind"] == "route":
        z = s.logits.to(f64)
        at = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :c["k"]]
        member = torch.zeros_like(z).scatter_(1, at, 1.0)
        p = torch.nan_to_num(torch.softmax(torch.where((member > 0) | (not c["normalize"]), z, -math.inf), dim=1), nan=0.0)
        weights = p.gather(1, at)
        out = [weights, None, None, None, None]
        if train:
            g = torch.zeros_like(z).scatter_(1, at, s.grad.to(f64))
            out.append(p * (g - (p * g).sum(dim=1, keepdim=True)))
        return out
    if c["kind"] == "exchange":
        n, k = c["tokens"], c["k"]
        x, y, w = s.x.to(f64), s.y.to(f64), s.weights.to(f64)
        token = torch.div(s.order, k, rounding_mode="floor").long()
        slot_weight = w.reshape(-1).index_select(0, s.order.long())[:, None]
        out = [x.index_select(0, token), torch.zeros_like(x).index_add_(0, token, y * slot_weight)]
        if train:
            g = s.grad.to(f64).index_select(0, token)
            dw = torch.zeros(n * k, device="cuda", dtype=f64)
            dw[s.order.long()] = (g * y).sum(dim=1)
            out += [torch.zeros_like(x).index_add_(0, token, s.grad_rows.to(f64)), g * slot_weight, dw.reshape(n, k)]
        return out
    bounds = s.offsets.tolist()
    y = torch.empty((c["rows"], c["n_out"]), device="cuda", dtype=f64)
    dx = torch.empty((c["rows"], c["n_in"]), device="cuda", dtype=f64) if train else None
    dw, db = [], []
    for e in range(c["experts"]):
        rows = slice(bounds[e], bounds[e + 1])
        x, w = s.x[rows].to(f64), s.weight[e].to(f64)
        y[rows] = x @ w.T + (s.bias[e].to(f64) if c["bias"] else 0.0)
        if train:
            g = s.grad[rows].to(f64)
            dx[rows] = g @ w
            dw.append(g.T @ x)
            db.append(g.sum(dim=0))
    if not train:
        return [y]
    return [y, dx, torch.stack(dw)] + ([torch.stack(db)] if c["bias"] else [])
