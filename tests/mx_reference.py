"""Dropout's generator and the 4-bit format from their definitions: Philox4x32-10 in numpy's integers, blocks in 64 bits."""
import numpy as np
import torch

from rows_reference import F64, sum_slack

LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def philox(counter, key):
    """four words (uint64 arrays of 32-bit values) of counters of four words and a key of two"""
    c, k = [np.asarray(v, dtype=np.uint64) for v in counter], [np.uint64(v) for v in key]
    low, shift = np.uint64(0xffffffff), np.uint64(32)
    for _ in range(10):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> shift) ^ c[1] ^ k[0], b & low, (a >> shift) ^ c[3] ^ k[1], a & low]
        k = [(k[0] + np.uint64(0x9E3779B9)) & low, (k[1] + np.uint64(0xBB67AE85)) & low]
    return c


def kept(first, n, p, seed, offset):
    """whether elements first .. first + n are kept; seed and offset modulo 2^64"""
    seed, offset = seed % 2 ** 64, offset % 2 ** 64
    i = np.arange(first, first + n, dtype=np.uint64)
    group = i // np.uint64(8)
    words = np.stack(philox([group & np.uint64(0xffffffff), group >> np.uint64(32), np.full_like(group, offset & 0xffffffff), np.full_like(group, offset >> 32)],
                            [seed & 0xffffffff, seed >> 32]), axis=1)
    at = (i % np.uint64(8)).astype(np.int64)
    numbers = words[np.arange(n), at // 2] >> (np.uint64(16) * (at % 2).astype(np.uint64)) & np.uint64(0xffff)
    return torch.from_numpy(numbers.astype(np.int64) >= round(p * 65536))


def dropout(x, keep, p, residual=None):
    """[(result, slack)]: a product with the rounded factor and a sum in fp32, before the last rounding"""
    cut = round(p * 65536)
    scaled = torch.where(keep, x.to(F64) * (65536 / max(1, 65536 - cut)), 0.0)
    r = torch.zeros_like(scaled) if residual is None else residual.to(F64)
    return scaled + r, 2.0 ** -23 * 1.01 * (scaled.abs() + (scaled + r).abs() + 2.0 ** -126)


def power_of_two(exponent):
    """exactly, from the bits of a 64-bit number"""
    return (exponent.long() + 1023 << 52).view(F64)


def quantize(x):
    """codes' numbers 0 .. 15 (..., blocks, 32) and exponents + 127 (..., blocks), by search for the nearest level"""
    n = x.shape[-1]
    x = torch.nn.functional.pad(x.to(F64), (0, -n % 32)).unflatten(-1, (-1, 32))
    finite = torch.isfinite(x).all(-1)
    clean = torch.where(finite[..., None], x, 0.0)
    largest = clean.abs().amax(-1)
    power = torch.where(largest > 0, torch.frexp(largest).exponent.to(torch.int64) - 3, -127).clamp(min=-127)
    at = clean.abs() * power_of_two(-power)[..., None]
    levels = torch.tensor(LEVELS, dtype=F64, device=x.device)
    distance = (at[..., None] - levels).abs()
    nearest = distance.amin(-1, keepdim=True)
    candidates = distance == nearest                                  # two at a tie: the even one
    order = torch.arange(8, device=x.device)
    number = torch.where(candidates, order + 8 * (order % 2), 100).amin(-1) % 8
    number = torch.where(at > 6, 7, number) + 8 * torch.signbit(clean).long()
    return number.to(torch.uint8), torch.where(finite, power + 127, 255).to(torch.uint8)


def values(number, exponent):
    levels = torch.tensor(LEVELS, dtype=F64, device=number.device)
    magnitude = levels[(number & 7).long()]
    scale = power_of_two(exponent.long() - 127)
    scale = torch.where(exponent == 255, float("nan"), scale)
    return (torch.where(number >= 8, -magnitude, magnitude) * scale[..., None]).flatten(-2)


def nearest(x):
    return values(*quantize(x))[..., :x.shape[-1]]


def pack(number, exponent):
    """the arrays of qmlp.MXTensor, entry by entry where they belong"""
    rows, blocks = exponent.shape[-2:]
    lead = exponent.shape[:-2]
    flat = number.flatten(-2).int()
    codes = (flat[..., 0::2] + 16 * flat[..., 1::2]).to(torch.uint8)
    scales = torch.zeros((*lead, (rows + 127) // 128, (blocks + 3) // 4, 32, 4, 4), dtype=torch.uint8, device=number.device)
    r, b = torch.meshgrid(torch.arange(rows, device=number.device), torch.arange(blocks, device=number.device), indexing="ij")
    scales[..., r // 128, b // 4, r % 32, r % 128 // 32, b % 4] = exponent
    return codes, scales


def bounds(offsets, rows, experts):
    b = [0, rows] if offsets is None else [min(max(int(o), 0), rows) for o in offsets]
    for i in range(1, len(b)):
        b[i] = max(b[i], b[i - 1])
    return b


def mx_linear(x, w, offsets, bias, grad=None):
    """[(result, slack)] of the output and, with `grad`, of the gradients of x and bias. w: (experts, channels out, channels in) values of a 4-bit tensor"""
    e, n_out, n_in = w.shape
    b = bounds(offsets, x.shape[0], e)
    y, ys = (torch.zeros((x.shape[0], n_out), dtype=F64, device=x.device) for _ in range(2))
    dx, dxs = (torch.zeros((x.shape[0], n_in), dtype=F64, device=x.device) for _ in range(2))
    db, dbs = (torch.zeros((e, n_out), dtype=F64, device=x.device) for _ in range(2))
    for i in range(e):
        r = slice(b[i], b[i + 1])
        q = nearest(x[r])
        shift = bias.view(e, n_out)[i].to(F64) if bias is not None else torch.zeros(n_out, dtype=F64, device=x.device)
        y[r] = q @ w[i].T + shift
        ys[r] = sum_slack(n_in, q.abs() @ w[i].abs().T + shift.abs())
        if grad is not None:
            g = grad[r].to(F64)
            dx[r], dxs[r] = g @ w[i], sum_slack(n_out, g.abs() @ w[i].abs())
            db[i], dbs[i] = g.sum(0), sum_slack(b[i + 1] - b[i], g.abs().sum(0))
    return [(y, ys)] + ([(dx, dxs), (db, dbs)] if grad is not None else [])
