"""The operators on feature rows in 64 bits, written from their definitions, with bounds on what 32-bit sums may lose.

A result is held to half a unit of its type's last place plus `slack`, the bound on the error before that rounding: a sum of n
terms in fp32, in any order, is off by at most n * 2^-23 times the sum of the terms' magnitudes (2^-23 per addition also covers sums
that are cut off instead of rounded, as a tensor core's may be)."""
import torch

F64 = torch.float64
HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}


def check(actual, exact, slack, name):
    """every entry within half a unit in the last place of the (slack-wide) exact value"""
    assert actual.shape == exact.shape, (name, actual.shape, exact.shape)
    a = actual.to(F64)
    fine = torch.isfinite(exact)
    assert torch.equal(torch.isnan(a), torch.isnan(exact)), name + ": NaN in other places"
    assert torch.equal(a[~fine & ~torch.isnan(exact)], exact[~fine & ~torch.isnan(exact)]), name + ": other infinities"
    bound = HALF_ULP[actual.dtype] * 1.001 * (exact.abs() + slack) + slack + TINY[actual.dtype]
    bad = ((a - exact).abs() > bound) & fine
    if bad.any():
        at = tuple(int(i) for i in bad.nonzero()[0])
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} entries off, first at {at}: {float(a[at])} for {float(exact[at])}, "
                             f"bound {float(torch.as_tensor(bound).expand_as(exact)[at])}")


def sum_slack(n, magnitude):
    return (n + 4) * 2.0 ** -23 * magnitude


def layer_norm(x, weight, bias, eps, grad=None):
    """[(result, slack)] of the output and, with `grad`, of the gradients of x, weight and bias"""
    x, c = x.to(F64), x.shape[-1]
    one = torch.ones(c, dtype=F64, device=x.device)
    w = one if weight is None else weight.to(F64)
    b = 0 * one if bias is None else bias.to(F64)
    mean = x.mean(-1, keepdim=True)
    d = x - mean
    sigma = ((d * d).mean(-1, keepdim=True) + eps).sqrt()
    u = d / sigma
    # the mean and the centred values in fp32; what they are off by enters the variance in the second order and through the sum
    du = sum_slack(c, (x.abs().mean(-1, keepdim=True) + x.abs()) / sigma) + sum_slack(c, u.abs()) + sum_slack(c, (x.abs().mean(-1, keepdim=True) / sigma)) * u.abs()
    out = [(u * w + b, du * w.abs() + 2.0 ** -22 * ((u * w).abs() + b.abs()))]
    if grad is None:
        return out
    g = grad.to(F64)
    gw = g * w
    m0, m1 = gw.mean(-1, keepdim=True), (gw * u).mean(-1, keepdim=True)
    dx = (gw - m0 - u * m1) / sigma
    size = gw.abs() + gw.abs().mean(-1, keepdim=True) + u.abs() * (gw * u).abs().mean(-1, keepdim=True)
    slack = (sum_slack(c, size) + du * m1.abs() + u.abs() * (gw.abs() * du).mean(-1, keepdim=True)) / sigma
    slack = slack + dx.abs() * sum_slack(c, 1.0) + dx.abs() * sum_slack(c, (x.abs().mean(-1, keepdim=True) / sigma))
    rows = x.shape[0]
    out.append((dx, slack))
    out.append(((g * u).sum(0), (g.abs() * du).sum(0) + sum_slack(rows, (g * u).abs().sum(0))))
    out.append((g.sum(0), sum_slack(rows, g.abs().sum(0))))
    return out


def embedding(tokens, table, scale, grad=None):
    v = table.shape[0]
    inside = (tokens >= 0) & (tokens < v)
    padded = torch.cat([table.to(F64), torch.zeros((1, table.shape[1]), dtype=F64, device=table.device)])
    at = torch.where(inside, tokens.long(), v)
    y = padded[at] * scale
    out = [(y, 2.0 ** -23 * y.abs())]
    if grad is not None:
        g = grad.to(F64).reshape(-1, table.shape[1])
        count = torch.bincount(at.reshape(-1), minlength=v + 1)[:v, None]
        total = torch.zeros_like(padded).index_add_(0, at.reshape(-1), g)[:v] * scale
        size = torch.zeros_like(padded).index_add_(0, at.reshape(-1), g.abs())[:v] * abs(scale)
        out.append((total, sum_slack(count, size)))
    return out


def route(logits, k, normalize):
    """weights, experts, order, positions, offsets; plain loops over the rows"""
    n, e = logits.shape
    z = logits.to(F64).cpu()
    weights, experts = torch.zeros((n, k), dtype=F64), torch.full((n, k), -1, dtype=torch.int32)
    for t in range(n):
        row = [float(v) for v in z[t]]
        choice = sorted((i for i in range(e) if row[i] != float("-inf")), key=lambda i: (row[i] == row[i], -row[i] if row[i] == row[i] else 0.0, i))[:k]
        if not choice:
            continue
        experts[t, :len(choice)] = torch.tensor(choice, dtype=torch.int32)
        over = z[t][choice] if normalize else z[t]
        share = torch.softmax(over, 0)
        weights[t, :len(choice)] = share[:len(choice)] if normalize else share[choice]
    flat = experts.reshape(-1)
    order = torch.full((n * k,), -1, dtype=torch.int32)
    positions = torch.full((n * k,), -1, dtype=torch.int32)
    offsets = torch.zeros(e + 1, dtype=torch.int32)
    at = 0
    for i in range(e):
        offsets[i] = at
        for s in (flat == i).nonzero().reshape(-1).tolist():
            order[at], positions[s] = s, at
            at += 1
    offsets[e] = at
    return weights, experts, order, positions.reshape(n, k), offsets


def route_gradient(logits, experts, weights, grad, normalize):
    """of the weights by the logits, from the definition of the softmax"""
    z, n, e = logits.to(F64), *logits.shape
    k = experts.shape[1]
    member = torch.zeros((n, e), dtype=torch.bool, device=z.device)
    g = torch.zeros_like(z)
    used = experts >= 0
    row = torch.arange(n, device=z.device)[:, None].expand(n, k)
    member[row[used], experts[used].long()] = True
    g[row[used], experts[used].long()] = grad.to(F64)[used]
    p = torch.softmax(torch.where(member, z, float("-inf")) if normalize else z, 1)
    p = torch.where((z != float("-inf")).any(1, keepdim=True), p, 0.0)
    inner = (p * g).sum(1, keepdim=True)
    size = p * (g.abs() + (p * g).abs().sum(1, keepdim=True))
    return p * (g - inner), sum_slack(e + 16, size)


def expert_linear(x, weight, offsets, bias, grad=None):
    """[(result, slack)] of the output and, with `grad`, of the gradients of x, weight and bias"""
    e, n_out, n_in = weight.shape
    bounds = [min(max(int(o), 0), x.shape[0]) for o in offsets]
    for i in range(1, len(bounds)):
        bounds[i] = max(bounds[i], bounds[i - 1])
    x, w = x.to(F64), weight.to(F64)
    y, ys = torch.zeros((x.shape[0], n_out), dtype=F64, device=x.device), torch.zeros((x.shape[0], n_out), dtype=F64, device=x.device)
    dx, dxs = torch.zeros_like(x), torch.zeros_like(x)
    dw, dws, db, dbs = torch.zeros_like(w), torch.zeros_like(w), torch.zeros((e, n_out), dtype=F64, device=x.device), torch.zeros((e, n_out), dtype=F64, device=x.device)
    for i in range(e):
        r = slice(bounds[i], bounds[i + 1])
        b = bias[i].to(F64) if bias is not None else torch.zeros(n_out, dtype=F64, device=x.device)
        y[r] = x[r] @ w[i].T + b
        ys[r] = sum_slack(n_in, x[r].abs() @ w[i].abs().T + b.abs())
        if grad is not None:
            g, rows = grad[r].to(F64), bounds[i + 1] - bounds[i]
            dx[r], dxs[r] = g @ w[i], sum_slack(n_out, g.abs() @ w[i].abs())
            dw[i], dws[i] = g.T @ x[r], sum_slack(rows, g.abs().T @ x[r].abs())
            db[i], dbs[i] = g.sum(0), sum_slack(rows, g.abs().sum(0))
    return [(y, ys)] + ([(dx, dxs), (dw, dws), (db, dbs)] if grad is not None else [])
