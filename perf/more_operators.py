"""Dropout and 4-bit layers on feature rows as measurable cases: what a program holds before the call (`prepare`), one pass
through the public entry points (`run` with `own`) or through elementary torch operations in 32 bits (`run` without), the
work a pass cannot do without (`work`) and its result in 64 bits (`exact`).

Kinds of cases (direction "forward": the result; "train": the result and the gradients of all that can have one)
  dropout  qmlp.dropout: rows with elements dropped by a counter-based generator (Philox4x32-10), alone or added to a residual
  mx       qmlp.mx_quantize and qmlp.mx_dequantize: rows to microscaled 4-bit floating point (blocks of 32 e2m1 elements with a
           power of two) and back
  linear   qmlp.mx_linear: products of rows, quantised in the call, with 4-bit matrices: one matrix, or one per expert
"""
import math
import os
import sys
from types import SimpleNamespace

import torch

own = False

DTYPES = {"float": torch.float32, "half": torch.float16, "bfloat16": torch.bfloat16}
BYTES = {"float": 4, "half": 2, "bfloat16": 2}
BLOCK = 32                      # channels that share a scale
MX_BYTES = 0.5 + 1 / BLOCK      # of an element


def _qmlp():
    path = os.path.abspath("quick-mlp_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import qmlp
    return qmlp


def listed():
    return [
        # the hidden rows of one interactive training step on a handful of points, where only latency counts
        dict(name="dropout_train_16x64", kind="dropout", direction="train", dtype="half", rows=16, channels=64, p=0.1, residual=False),
        # the hidden rows of a batch of a million points in a narrow network
        dict(name="dropout_train_1mx64", kind="dropout", direction="train", dtype="half", rows=1000003, channels=64, p=0.1, residual=False),
        # rows of an odd width in full precision, added to what they were computed from
        dict(name="dropout_train_100kx77_float", kind="dropout", direction="train", dtype="float", rows=100003, channels=77, p=0.5, residual=True),
        # the activations of a wide model over a large batch, added to the residual stream
        dict(name="dropout_train_32kx4096", kind="dropout", direction="train", dtype="bfloat16", rows=32768, channels=4096, p=0.1, residual=True),
        # one latent code kept in 4 bits
        dict(name="mx_1x1024", kind="mx", direction="forward", dtype="half", rows=1, channels=1024, relu=False),
        # a table of codes of an odd width in full precision
        dict(name="mx_20kx777_float", kind="mx", direction="forward", dtype="float", rows=20011, channels=777, relu=False),
        # the activations of a large batch behind a relu, kept in 4 bits and read back
        dict(name="mx_128kx1024", kind="mx", direction="forward", dtype="bfloat16", rows=131072, channels=1024, relu=True),
        # one query served by two experts of 64
        dict(name="linear_forward_2", kind="linear", direction="forward", dtype="half", rows=2, experts=64, n_in=1024, n_out=2048, bias=True, spread=0.5),
        # one row through one wide matrix
        dict(name="linear_forward_1x4096x4096", kind="linear", direction="forward", dtype="bfloat16", rows=1, experts=0, n_in=4096, n_out=4096, bias=False,
             spread=0.0),
        # many small experts, each in charge of a part of the scene, a million points of a frame over them
        dict(name="linear_forward_1mx64x64", kind="linear", direction="forward", dtype="half", rows=1000003, experts=512, n_in=64, n_out=64, bias=True,
             spread=0.3),
        # what is in front of a wide layer of frozen 4-bit experts is trained
        dict(name="linear_train_128kx1024", kind="linear", direction="train", dtype="bfloat16", rows=131072, experts=16, n_in=1024, n_out=1024, bias=True,
             spread=0.3),
        # a batch through one wide matrix
        dict(name="linear_forward_16kx4096x4096", kind="linear", direction="forward", dtype="bfloat16", rows=16384, experts=0, n_in=4096, n_out=4096, bias=True,
             spread=0.0),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _size(rng, low, high, step):
    """spread over the logarithm; more than half are multiples of `step`, the rest whatever comes, odd ones among them"""
    n = _log(rng, low, high)
    return max(low, n // step * step) if rng.random() < 0.6 else n


def draw(rng):
    kind = rng.choice(["dropout", "dropout", "mx", "linear", "linear", "linear"])
    c = dict(kind=kind, direction="forward" if kind == "mx" else rng.choice(["forward", "train", "train"] if kind == "dropout" else ["forward", "forward", "train"]))
    if kind == "dropout":
        c["dtype"] = rng.choice(["half", "bfloat16", "float"])
        c["channels"] = _size(rng, 1, 16384, 8)
        c["rows"] = _log(rng, 1, max(1, min(1 << 20, (1 << 26) // c["channels"])))
        c["p"] = rng.choice([0.0, 0.05, 0.1, 0.25, 0.5, 0.9])
        c["residual"] = rng.random() < 0.5
    elif kind == "mx":
        c["dtype"] = rng.choice(["half", "bfloat16", "float"])
        c["channels"] = _size(rng, 1, 16384, 32)
        c["rows"] = _log(rng, 1, max(1, min(1 << 18, (1 << 26) // c["channels"])))
        c["relu"] = rng.random() < 0.3
    else:
        c["dtype"] = rng.choice(["half", "bfloat16"])
        c["experts"] = 0 if rng.random() < 0.4 else _log(rng, 1, 512)
        c["n_in"] = _size(rng, 8, 4096, 32)
        c["n_out"] = _size(rng, 8, max(16, min(4096, (1 << 25) // (c["n_in"] * max(1, c["experts"])))), 8)
        c["rows"] = _log(rng, 1, max(1, min(1 << 20, (1 << 37) // (c["n_in"] * c["n_out"]), (1 << 27) // (c["n_in"] + c["n_out"]))))
        c["bias"] = rng.random() < 0.7
        c["spread"] = rng.choice([0.0, 0.3, 0.6])
    return c


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _normal(gen, shape, dtype, std=1.0, mean=0.0):
    return (torch.randn(shape, device="cuda", generator=gen) * std + mean).to(DTYPES[dtype])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c, s = case, SimpleNamespace(case=case)
    train = c["direction"] == "train"
    if c["kind"] == "dropout":
        shape = (c["rows"], c["channels"])
        s.seed, s.offset = int(torch.randint(1 << 62, (1,), generator=torch.Generator().manual_seed(seed))), seed % 1000
        s.x = _normal(gen, shape, c["dtype"], 1.5)
        s.residual = _normal(gen, shape, c["dtype"]) if c["residual"] else None
        s.grad = _normal(gen, shape, c["dtype"]) if train else None
        leaves = [s.x, s.residual]
    elif c["kind"] == "mx":
        # rows of different magnitude
        scale = torch.exp(torch.randn((c["rows"], 1), device="cuda", generator=gen))
        x = torch.randn((c["rows"], c["channels"]), device="cuda", generator=gen) * scale
        s.x = (x.relu_() if c["relu"] else x).to(DTYPES[c["dtype"]])
        leaves = []
    else:
        e = max(1, c["experts"])
        popular = torch.exp(torch.randn(e, device="cuda", generator=gen) * c["spread"]).double().cpu()
        bounds = torch.round(c["rows"] * popular.cumsum(0) / popular.sum()).int()
        s.offsets = torch.nn.functional.pad(bounds, (1, 0)).cuda() if c["experts"] else None
        s.most = int(torch.diff(bounds, prepend=bounds.new_zeros(1)).max())      # the plan of a program that pads to the longest run
        s.x = _normal(gen, (c["rows"], c["n_in"]), c["dtype"])
        weight = _normal(gen, (e, c["n_out"], c["n_in"]), "float", c["n_in"] ** -0.5)
        s.codes, s.scales = _pack(*_quantize(weight))
        if not c["experts"]:
            s.codes, s.scales = s.codes[0], s.scales[0]
        s.bias = _normal(gen, (e, c["n_out"]) if c["experts"] else (c["n_out"],), c["dtype"], 0.1) if c["bias"] else None
        s.grad = _normal(gen, (c["rows"], c["n_out"]), c["dtype"]) if train else None
        if own:
            s.weight = _qmlp().MXTensor(s.codes, s.scales, c["n_in"])
        leaves = [s.x, s.bias]
    if train:
        s.leaves = [t.requires_grad_() for t in leaves if t is not None]
    return s


# ---- one pass through the framework ----------------------------------------------------------------------------------
def _own_pass(s):
    qmlp, c = _qmlp(), s.case
    if c["kind"] == "dropout":
        y = qmlp.dropout(s.x, c["p"], s.seed, s.offset, residual=s.residual)
    elif c["kind"] == "mx":
        return [qmlp.mx_dequantize(qmlp.mx_quantize(s.x), s.x.dtype)]
    else:
        y = qmlp.mx_linear(s.x, s.weight, s.offsets, s.bias)
    if c["direction"] != "train":
        return [y]
    return [y.detach(), *torch.autograd.grad(y, s.leaves, s.grad)]


# ---- the plain forms: elementary operations in 32 bits, rounded once at the end ----------------------------------------
def _kept(n, p, seed, offset):
    """whether the first n elements are kept, in the order of the rows: 16 bits each of Philox4x32-10, eight elements a counter"""
    groups = torch.arange((n + 7) // 8, device="cuda")
    low = 0xffffffff
    c0, c1 = groups & low, groups >> 32
    c2, c3 = torch.full_like(groups, offset & low), torch.full_like(groups, offset >> 32 & low)
    k0, k1 = seed & low, seed >> 32 & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57     # (64-bit products wrap; the shift's sign is masked away)
        c0, c1, c2, c3 = (b >> 32 & low) ^ c1 ^ k0, b & low, (a >> 32 & low) ^ c3 ^ k1, a & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    words = torch.stack([c0, c1, c2, c3], dim=1)
    numbers = torch.stack([words & 0xffff, words >> 16], dim=2).reshape(-1)[:n]
    return numbers >= round(p * 65536)


def _plain_dropout(s, c, dtype):
    kept = _kept(s.x.numel(), c["p"], s.seed, s.offset).view(s.x.shape)
    scale = 65536 / (65536 - round(c["p"] * 65536))
    y = torch.where(kept, s.x.float() * scale, 0.0)
    out = [(y + s.residual.float() if c["residual"] else y).to(dtype)]
    if c["direction"] == "train":
        out.append(torch.where(kept, s.grad.float() * scale, 0.0).to(dtype))
        if c["residual"]:
            out.append(s.grad)
    return out


def _power(biased):
    """2 ** (biased - 127) in fp32, from its bits; the lowest is not a normal number"""
    return torch.where(biased == 0, 1 << 22, biased.int() << 23).int().view(torch.float32)


def _quantize(x):
    """(..., channels) -> magnitudes' numbers with signs (..., blocks, 32) uint8 and exponents + 127 (..., blocks)"""
    x = torch.nn.functional.pad(x.float(), (0, -x.shape[-1] % BLOCK)).unflatten(-1, (-1, BLOCK))
    bits = x.abs().amax(dim=-1).view(torch.int32) >> 23
    exponent = torch.where(bits == 255, 255, (bits - 2).clamp(min=0))
    at = x.abs() * _power((254 - exponent).clamp(min=0))[..., None]
    number = sum((at > m).to(torch.uint8) if down else (at >= m).to(torch.uint8)      # borders; a tie goes to the even number
                 for m, down in ((0.25, True), (0.75, False), (1.25, True), (1.75, False), (2.5, True), (3.5, False), (5.0, True)))
    return number + 8 * (x < 0).to(torch.uint8), exponent


def _values(number, exponent):
    """the numbers' values (..., channels up to a multiple of 32)"""
    level = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device="cuda")[(number & 7).int()]
    scale = torch.where(exponent == 255, math.nan, _power(exponent))
    return (torch.where(number >= 8, -level, level) * scale[..., None]).flatten(-2)


def _pack(number, exponent):
    """codes (..., rows, 16 * blocks): two elements a byte, the first in the low bits; scales (..., rows / 128, channels / 128, 32, 4, 4):
    [t, c, i, q, j] is that of row 128 t + 32 q + i and of the channels from 128 c + 32 j on"""
    flat = number.flatten(-2)
    rows, blocks = exponent.shape[-2:]
    tiles = torch.nn.functional.pad(exponent.to(torch.uint8), (0, -blocks % 4, 0, -rows % 128)).unflatten(-1, (-1, 4)).unflatten(-3, (-1, 4, 32))
    return flat[..., 0::2] | flat[..., 1::2] << 4, tiles.movedim(-2, -4).transpose(-2, -3).contiguous()


def _unpack(codes, scales):
    rows, blocks = codes.shape[-2], codes.shape[-1] // 16
    number = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).unflatten(-1, (-1, BLOCK))
    tiles = scales.transpose(-2, -3).movedim(-4, -2)
    return number, tiles.flatten(-2).flatten(-4, -2)[..., :rows, :blocks]


def _plain_mx(s, c, dtype):
    return [_values(*_quantize(s.x))[:, :c["channels"]].to(dtype)]


def _plain_linear(s, c, dtype):
    e = max(1, c["experts"])
    x = _values(*_quantize(s.x))[:, :c["n_in"]]
    rows = torch.arange(c["rows"], device="cuda")
    offsets = s.offsets.long() if c["experts"] else torch.tensor([0, c["rows"]], device="cuda")
    expert = torch.searchsorted(offsets[1:].contiguous(), rows, right=True)
    number, exponent = _unpack(s.codes.view(e, c["n_out"], -1), s.scales.view(e, *s.scales.shape[-5:]))
    bias = s.bias.float().view(e, -1) if c["bias"] else None
    if c["rows"] <= 64 and c["direction"] == "forward":     # few rows: each with its expert's matrix
        w = _values(number[expert], exponent[expert])[..., :c["n_in"]]
        y = torch.einsum("rk,rnk->rn", x, w)
        return [(y + bias[expert] if c["bias"] else y).to(dtype)]
    w = _values(number, exponent)[..., :c["n_in"]]
    slot = rows - offsets[expert]
    padded = x.new_zeros((e, s.most, c["n_in"]))
    padded[expert, slot] = x
    y = torch.bmm(padded, w.transpose(1, 2))[expert, slot]
    out = [(y + bias[expert] if c["bias"] else y).to(dtype)]
    if c["direction"] == "train":
        g = x.new_zeros((e, s.most, c["n_out"]))
        g[expert, slot] = s.grad.float()
        out.append(torch.bmm(g, w)[expert, slot].to(dtype))
        if c["bias"]:
            out.append(g.sum(dim=1).view(s.bias.shape).to(dtype))
    return out


PLAIN = {"dropout": _plain_dropout, "mx": _plain_mx, "linear": _plain_linear}


def run(state):
    if own:
        return _own_pass(state)
    with torch.no_grad():   # the plain forms write their gradients out
        return PLAIN[state.case["kind"]](state, state.case, DTYPES[state.case["dtype"]])


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    c, train = case, case["direction"] == "train"
    b = BYTES[c["dtype"]]
    if c["kind"] == "dropout":
        n = c["rows"] * c["channels"]
        return {"bytes": n * b * (2 + c["residual"] + (2 if train else 0)), "flops": n * (2 if train else 1)}
    if c["kind"] == "mx":
        n = c["rows"] * c["channels"]
        # in and out, and the 4-bit form written and read between
        return {"bytes": int(n * (2 * b + 2 * MX_BYTES)), "flops": n * 4}
    matrices = min(max(1, c["experts"]), c["rows"]) * c["n_in"] * c["n_out"]
    flops = 2 * c["rows"] * c["n_in"] * c["n_out"]
    forward = int(c["rows"] * (c["n_in"] + c["n_out"]) * b + matrices * MX_BYTES)
    if not train:
        return {"bytes": forward, "flops": flops}
    # dy in, dx out; the matrices were just read
    return {"bytes": forward + c["rows"] * (c["n_in"] + c["n_out"]) * b, "flops": 2 * flops}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def _philox_words(group, offset, seed):
    """Philox4x32-10 of one counter, in Python's integers: a check of the generator's first elements"""
    c, k = [group & 0xffffffff, group >> 32, offset & 0xffffffff, offset >> 32], [seed & 0xffffffff, seed >> 32]
    for r in range(10):
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 % 2 ** 32, (p0 >> 32) ^ c[3] ^ k[1], p0 % 2 ** 32]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return c


def _power64(exponent):
    return (exponent.long() + 1023 << 52).view(torch.float64)


def _nearest(x):
    """microscaled values of (..., channels) in 64 bits"""
    n = x.shape[-1]
    x = torch.nn.functional.pad(x.to(torch.float64), (0, -n % BLOCK)).unflatten(-1, (-1, BLOCK))
    power = torch.frexp(x.abs().amax(dim=-1, keepdim=True)).exponent - 3      # the largest is in [2^(power + 2), 2^(power + 3))
    unit = _power64(power.clamp(min=-127))
    a = x.abs() / unit
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return (torch.copysign(torch.clamp(torch.round(a / step) * step, max=6.0), x) * unit).flatten(-2)[..., :n]


@torch.no_grad()
def exact(case, seed):
    s, c, train = prepare(case, seed), case, case["direction"] == "train"
    f64 = torch.float64
    if c["kind"] == "dropout":
        cut = round(c["p"] * 65536)
        kept = _kept(s.x.numel(), c["p"], s.seed, s.offset)
        for group in (0, (s.x.numel() - 1) // 8):      # (the numbers are integers: what Python says of them has to be the same)
            words = _philox_words(group, s.offset, s.seed)
            expected = [(words[i // 2] >> 16 * (i % 2)) % 65536 >= cut for i in range(8)][:s.x.numel() - 8 * group]
            if kept[8 * group:8 * group + 8].tolist() != expected:
                raise RuntimeError("the generator's integers differ")
        keep = kept.view(s.x.shape).to(f64) / (1 - cut / 65536)
        out = [s.x.to(f64) * keep + (s.residual.to(f64) if c["residual"] else 0.0)]
        if train:
            out += [s.grad.to(f64) * keep] + ([s.grad.to(f64)] if c["residual"] else [])
        return out
    if c["kind"] == "mx":
        return [_nearest(s.x)]
    # the weights as prepared: bytes looked up, scales by their place
    e, n = max(1, c["experts"]), c["n_out"]
    codes, scales = s.codes.view(e, n, -1), s.scales.view(e, *s.scales.shape[-5:])
    level = [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    pair = torch.tensor([[(-1) ** (v >> 3) * level[v & 7] for v in (b & 15, b >> 4)] for b in range(256)], device="cuda", dtype=f64)
    row, block = torch.arange(n, device="cuda")[:, None], torch.arange(codes.shape[-1] // 16, device="cuda")[None]
    bounds = s.offsets.tolist() if c["experts"] else [0, c["rows"]]
    y = torch.empty((c["rows"], n), device="cuda", dtype=f64)
    dx = torch.empty((c["rows"], c["n_in"]), device="cuda", dtype=f64) if train else None
    db = []
    for i in range(e):
        power = scales[i][row // 128, block // 4, row % 32, row // 32 % 4, block % 4].int() - 127
        w = (pair[codes[i].int()].view(n, -1, BLOCK) * _power64(power)[..., None]).view(n, -1)[:, :c["n_in"]]
        rows = slice(bounds[i], bounds[i + 1])
        y[rows] = _nearest(s.x[rows]) @ w.T
        if c["bias"]:
            y[rows] += s.bias.view(e, n)[i].to(f64)
        if train:
            g = s.grad[rows].to(f64)
            dx[rows] = g @ w
            db.append(g.sum(dim=0))
    if not train:
        return [y]
    return [y, dx] + ([torch.stack(db).view(s.bias.shape)] if c["bias"] else [])
