"""The low-bit operators of an attention block from their definitions in 64
bits (torch, on the CPU), with the error that each kernel may have on top."""
import math

import torch

import operator_refs as ref

LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def turn(x, positions, freq, half, magnitude=1.0):
    """x [rows, heads, d] float64, turned."""
    r = 2 * len(freq)
    angle = positions.double()[:, None, None] * freq
    c, s = magnitude * angle.cos(), magnitude * angle.sin()
    first, second = (slice(0, r // 2), slice(r // 2, r)) if half else (slice(0, r, 2), slice(1, r, 2))
    y = x.clone()
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    return y


def head_norm(x, w, eps, positions, freq, half, magnitude):
    """x [rows, heads, d], w [d] or [heads, d] or None -> normed and turned,
    with tolerances. A lane adds at most 16 squares and exchanges 6 times, which
    the root halves: 11 2^-24; the mean, epsilon, root, quotient and two
    products round once each. The rotation's own error as in
    operator_refs.rope."""
    x = x.double()
    h = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if w is not None:
        h = h * w.double()
    y = turn(h, positions, freq, half, magnitude)
    r = 2 * len(freq)
    first = slice(0, r // 2) if half else slice(0, r, 2)
    second = slice(r // 2, r) if half else slice(1, r, 2)
    both = h.abs().clone()
    pair = abs(magnitude) * (h[..., first].abs() + h[..., second].abs())
    both[..., first] = both[..., second] = pair
    far = torch.zeros_like(both)
    far[..., first] = far[..., second] = 2.0 ** -51 * positions.double().abs()[:, None, None] * freq
    return y, both * ((17 + 12) * 2.0 ** -24 + far)


def matmul8(x, xs, w, ws, bias, dtype):
    """The sum, exact; its rounding to 32 bits, two products, the bias's
    addition and the rounding to the type."""
    y = (x.double() @ w.double().T) * xs.double()[:, None] * ws.double()
    mag = y.abs()
    if bias is not None:
        y = y + bias.double()
        mag = mag + bias.double().abs()
    return y, ref.HALF[dtype] * y.abs() + 5 * 2.0 ** -24 * mag + ref.TINY[dtype]


def encode4(x):
    """x [..., D] float64 -> codes and scale bytes by the definition, and how
    near a value is to another code, relative to its block's power of two."""
    blocks = x.unflatten(-1, (-1, 32))
    peak = blocks.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(blocks).all(-1, keepdim=True)
    s = torch.full(peak.shape, -126.0, dtype=torch.float64)
    for e in range(-126, 126):  # the smallest with peak <= 7 2^s
        s = torch.where((peak > 7 * 2.0 ** e) & (s == e), s + 1, s)
    s = s.clamp(max=125)
    u = torch.where(bad, torch.zeros_like(blocks), blocks / 2.0 ** s)
    dist = (u.abs()[..., None] - torch.tensor(LEVELS, dtype=torch.float64)).abs()
    best = dist.amin(-1, keepdim=True)
    near = dist == best  # two on a tie: the even code
    codes = torch.where(near[..., 0::2].any(-1), near[..., 0::2].int().argmax(-1) * 2, near[..., 1::2].int().argmax(-1) * 2 + 1)
    codes = codes + 8 * torch.signbit(u).long()
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
    margin = (u.abs()[..., None] - borders).abs().amin(-1)
    bytes_ = torch.where(bad, torch.full_like(s, 255.0), s + 127).squeeze(-1).to(torch.uint8)
    return codes.flatten(-2).to(torch.uint8), bytes_, margin.flatten(-2)


def decode4(codes, scales):
    """Values [..., D] of codes and scale bytes [..., D / 32]."""
    levels = torch.tensor(LEVELS + [-v for v in LEVELS], dtype=torch.float64)
    v = levels[codes.long()].unflatten(-1, (-1, 32))
    p = torch.where(scales == 255, torch.full(scales.shape, math.nan, dtype=torch.float64),
                    2.0 ** (scales.double() - 127))
    return (v * p[..., None]).flatten(-2)


def pack_pages(kc, ks, vc, vs, page):
    """Codes [tokens, heads, D] and scales [tokens, heads, D / 32] of a whole
    number of pages -> bytes [pages, heads * page * (D + D / 16)]."""
    T, H, D = kc.shape
    N = T // page
    parts = []
    for codes, value in ((kc, False), (vc, True)):
        two = (codes[..., 0::2] | (codes[..., 1::2] << 4)).view(N, page, H, D // 2).transpose(1, 2)
        if value:  # token of four behind the piece
            two = two.reshape(N, H, page // 4, 4, 16, D // 32).permute(0, 1, 2, 4, 3, 5)
        parts.append(two.reshape(N, H, -1))
    for scales in (ks, vs):
        parts.append(scales.view(N, page // 8, 8, H, D // 32).permute(0, 3, 1, 4, 2).reshape(N, H, -1))
    return torch.cat(parts, -1).reshape(N, -1)
