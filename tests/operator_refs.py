"""The attention block's operators from their definitions in 64 bits (torch,
on the CPU), with the error that each kernel may have on top: one rounding of
a result to a type is off by at most eps(type) / 2 of it, sums of n products in
32 bits by n 2^-24 of the sum of magnitudes."""
import math

import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
# half the smallest step below the normal range
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


def rope_frequencies(rotary, theta, scaling="none", factor=1.0, original=16384, fast=32.0, slow=1.0, low=1.0,
                     high=4.0):
    f = []
    for i in range(rotary // 2):
        base = theta ** (-2.0 * i / rotary)
        if scaling == "linear":
            base /= factor
        elif scaling == "yarn":
            def pair_of(turns):
                return rotary * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))
            a, b = max(0, math.floor(pair_of(fast))), min(rotary - 1, math.ceil(pair_of(slow)))
            ramp = min(1.0, max(0.0, (i - a) / max(0.001, b - a)))
            base = ramp * base / factor + (1 - ramp) * base
        elif scaling == "bands":
            turns = original * base / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - low) / (high - low)))
            base = (1 - keep) * base / factor + keep * base
        f.append(base)
    return torch.tensor(f, dtype=torch.float64)


def rope(x, positions, freq, half, magnitude=1.0):
    """x [rows, heads, d] -> its rotation and the tolerance of each value."""
    r = 2 * len(freq)
    angle = positions.double()[:, None, None] * freq
    c, s = magnitude * angle.cos(), magnitude * angle.sin()
    first = slice(0, r // 2) if half else slice(0, r, 2)
    second = slice(r // 2, r) if half else slice(1, r, 2)
    y = x.double().clone()
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    # two products, a sum, the sine's and cosine's own error (a few 2^-24) and
    # that of the angle's remainder (2 pi 2^-25) and, for far positions, of the
    # angle itself (2^-52 of it)
    far = 2.0 ** -51 * (positions.double().abs()[:, None, None] * freq)
    slack = torch.zeros_like(y)
    slack[..., first] = slack[..., second] = (abs(magnitude) * (12 * 2.0 ** -24 + far)) * (a.abs() + b.abs())
    exact = torch.zeros_like(y, dtype=torch.bool)
    exact[..., r:] = True
    tol = HALF[x.dtype] * y.abs() + slack + TINY[x.dtype]
    return y, torch.where(exact, torch.zeros_like(tol), tol)


def norm(x, delta, w, eps):
    """h and y in 64 bits, and the relative error that 32-bit sums leave on y:
    a value's square and the 2 hidden / 64 + 16 additions after it are in
    32 bits, the root halves that; h, 1 / root and two products round once
    each."""
    h = x.double() + (delta.double() if delta is not None else 0)
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * (w.double() if w is not None else 1)
    return h, y, (h.shape[-1] / 64 + 16) * 2.0 ** -24


def visible(queries, keys, left, right, sinks):
    """[queries, keys]: which key each query sees."""
    p = (torch.arange(queries) + keys - queries)[:, None]
    j = torch.arange(keys)[None, :]
    see = torch.ones(queries, keys, dtype=torch.bool)
    if right >= 0:
        see &= j <= p + right
    if left >= 0:
        see &= (j >= p - left) | (j < sinks)
    return see


def attention(q, k, v, left, right, sinks, scale):
    """q [n, H, D], k and v [m, K, D] -> out [n, H, D] and its tolerance.

    A score is D products summed in 32 bits and scaled; its error is the
    probability's relative error, twice (the sum over the probabilities has
    it too). Probabilities are rounded to the type before the product with v,
    which sums in 32 bits; the output is rounded once.

    Half precision's probabilities below 2^-14 are rounded by up to 2^-25
    whatever they are: the kernels take them against the row's largest score
    at the time, whose own is 1, so their sum is at least 1 and the n seen
    keys add 2^-25 (sum |v| + n |out|)."""
    n, H, D = q.shape
    m, K = k.shape[0], k.shape[1]
    out = torch.zeros(n, H, D, dtype=torch.float64)
    tol = torch.zeros_like(out)
    see = visible(n, m, left, right, sinks)
    if n == 0 or m == 0:
        return out, tol
    hidden = ~see
    for h in range(H):
        kk, vv = k[:, h * K // H].double(), v[:, h * K // H].double()
        # keys that no query sees may hold anything
        gone = ~see.any(0)
        kk, vv = kk.clone(), vv.clone()
        kk[gone] = 0
        vv[gone] = 0
        qq = q[:, h].double()
        s = (qq @ kk.T * scale).masked_fill(hidden, -math.inf)
        mag = (qq.abs() @ kk.abs().T * scale).masked_fill(hidden, 0).amax(-1, keepdim=True)
        p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
        out[:, h] = p @ vv
        weight = p @ vv.abs()
        err = 2 * mag * (D + 4) * 2.0 ** -24 + HALF[q.dtype] + (m / 16 + 32) * 2.0 ** -24
        tol[:, h] = weight * err + HALF[q.dtype] * out[:, h].abs() + TINY[q.dtype]
        seen = see.double()
        tol[:, h] += TINY[q.dtype] * (seen @ vv.abs() + seen.sum(1, keepdim=True) * out[:, h].abs())
    return out, tol
