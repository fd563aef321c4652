"""What the speed of the attention block's operators is measured on: rotary
positions, attention with a sliding window and sinks, and the residual
RMSNorm with 8-bit output, each in a plain form of elementary torch
operations and through the package's kernels, with inputs made from a seed
alone and 64-bit results.

Queries, keys, values, hidden states and residuals are N(0, 1), norm weights
N(1, 0.1).
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PACKAGE = os.path.join(_ROOT, "nemotron-3-embed-webgpu_amd")

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
EPS = 1e-5
CHUNK = 256  # queries of a block of the plain attention


def _rope(name, type_, rows, heads, kv_heads, head_dim, rotary, layout, scaling, theta, far):
    c = {"op": "rope", "type": type_, "rows": rows, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
         "rotary": rotary, "layout": layout, "scaling": scaling, "theta": theta, "far": far}
    return dict(c, name=name) if name else c


def _norm(name, type_, rows, hidden, type8, group, both):
    c = {"op": "norm", "type": type_, "rows": rows, "hidden": hidden, "type8": type8, "group": group, "both": both}
    return dict(c, name=name) if name else c


def _attention(name, type_, heads, kv_heads, head_dim, left, right, sinks, q_lens, kv_lens):
    """kv_lens None: a packed batch whose rows hold query, key and value heads; else a cache of each request's rows."""
    c = {"op": "attention", "type": type_, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "left": left,
         "right": right, "sinks": sinks, "q_lens": ",".join(map(str, q_lens)),
         "kv_lens": ",".join(map(str, kv_lens)) if kv_lens else ""}
    return dict(c, name=name) if name else c


# a micro-batch of queries and passages of mixed lengths
RAGGED = [15, 15, 50, 50, 150, 150, 500, 500, 15, 50, 150, 500, 15, 50, 150, 500]
# how far 64 conversations have come
CACHED = [97 + (i * i * 7919 + 613 * i) % 32600 for i in range(64)]


def listed():
    return [
        # one token's query and key heads, as each step of a decoder turns them
        _rope("rope_1_token", "f16", 1, 32, 8, 64, 64, "interleaved", "yarn", 1e6, 5000),
        # a page of float32 heads of which a part is turned: odd counts, pairs half the turned part apart
        _rope("rope_5001_partial", "f32", 5001, 12, 3, 96, 40, "half", "linear", 1e4, 5001),
        # a long document's heads at far positions
        _rope("rope_32768_far", "bf16", 32768, 32, 8, 128, 128, "half", "bands", 5e5, 1 << 20),
        # one token's hidden state between attention and FFN
        _norm("norm_1x2048", "f16", 1, 2048, "i8", 0, False),
        # one short of a benchmark batch: token states for an index, one scale a token
        _norm("norm_2399x2048", "f16", 2399, 2048, "i8", 0, True),
        # a long document, wide states, block scales for 8-bit products
        _norm("norm_16384x8192", "bf16", 16384, 8192, "e4m3", 128, False),
        # one conversation's next token: the smallest attention
        _attention("attention_1_token", "f16", 32, 8, 64, 1023, 0, 4, [1], [5000]),
        # the next token of 64 conversations of all lengths
        _attention("attention_64_tokens", "bf16", 32, 8, 128, 4095, 0, 4, [1] * 64, CACHED),
        # the next token of one long document, every key visible
        _attention("attention_1_token_all", "bf16", 32, 8, 128, -1, 0, 0, [1], [131072]),
        # a micro-batch through an encoder with local layers
        _attention("attention_ragged16", "f16", 32, 8, 64, 128, 128, 0, RAGGED, None),
        # prompts arriving in pieces behind what is cached
        _attention("attention_pieces", "f16", 16, 4, 128, 1023, 0, 16, [512, 77, 1, 300], [9000, 77, 4097, 1300]),
        # a long document's prompt
        _attention("attention_32768", "bf16", 32, 8, 128, 1023, 0, 4, [32768], None),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "norm", "attention", "attention"])
    if op == "rope":
        head_dim = rng.choice([64, 64, 80, 96, 128, 128])
        rotary = head_dim if rng.random() < 0.6 else 2 * rng.randint(4, head_dim // 2)
        kv_heads = rng.choice([1, 2, 3, 8])
        return _rope("", rng.choice(["f16", "bf16", "f32"]), _log_int(rng, 1, 8192), kv_heads * rng.choice([1, 3, 4]),
                     kv_heads, head_dim, rotary, rng.choice(["interleaved", "half"]),
                     rng.choice(["none", "linear", "yarn", "bands"]), rng.choice([1e4, 5e5, 1e6]),
                     _log_int(rng, 1, 1 << 24))
    if op == "norm":
        hidden, group = _log_int(rng, 64, 8192), 0
        if rng.random() < 0.7:
            group = rng.choice([0, 32, 64, 128])
            hidden = max(128, hidden // 128 * 128)
        return _norm("", rng.choice(["f16", "bf16", "f32"]), _log_int(rng, 1, 8192), hidden,
                     rng.choice(["i8", "e4m3"]), group, rng.random() < 0.5)
    head_dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * min(rng.choice([1, 2, 3, 4, 5, 8]), 32 // kv_heads)
    type_ = rng.choice(["f16", "bf16"])
    left = rng.choice([-1, _log_int(rng, 1, 2048) - 1, _log_int(rng, 64, 2048)])
    sinks = rng.choice([0, 0, 1, 4, 100])
    count = rng.randint(1, 8)
    if rng.random() < 0.5:  # packed: encoders and prompts
        lens = [_log_int(rng, 1, 1500) for _ in range(count)]
        right = rng.choice([0, 0, -1, _log_int(rng, 1, 512)])
        return _attention("", type_, heads, kv_heads, head_dim, left, right, sinks, lens, None)
    one = rng.random() < 0.5
    lens = [1 if one else _log_int(rng, 1, 200) for _ in range(count)]
    return _attention("", type_, heads, kv_heads, head_dim, left, 0, sinks, lens,
                      [n + _log_int(rng, 1, 32000 if one else 12000) - 1 for n in lens])


def _ints(text):
    return [int(t) for t in text.split(",")]


def _positions(case):
    """Rows that run on to the far end, or, where that is far behind them, rows spread over the way to it."""
    rows = case["rows"]
    return (torch.arange(rows, dtype=torch.int64) * 7919 % max(1, case["far"])) if rows * 4 < case["far"] else (
        torch.arange(rows, dtype=torch.int64) + max(0, case["far"] - rows))


def prepare(case, seed):
    """Inputs on the GPU, outputs' buffers and, for the package's kernels, the handle that a program keeps."""
    g = torch.Generator(device="cuda")
    g.manual_seed(1 + int(seed))
    dt = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dt)

    s = {"case": case}
    if case["op"] == "rope":
        rows, hd = case["rows"], case["head_dim"]
        s["q"], s["k"] = normal(rows, case["heads"], hd), normal(rows, case["kv_heads"], hd)
        s["positions"] = (_positions(case) + int(seed) % 7).cuda()
    elif case["op"] == "norm":
        s["x"], s["delta"] = normal(case["rows"], case["hidden"]), normal(case["rows"], case["hidden"])
        s["w"] = 1 + 0.1 * torch.randn(case["hidden"], generator=g, device="cuda", dtype=torch.float32)
    else:
        H, K, D = case["heads"], case["kv_heads"], case["head_dim"]
        lens = _ints(case["q_lens"])
        rows = sum(lens)
        s["q_lens"] = lens
        if case["kv_lens"]:
            s["kv_lens"] = _ints(case["kv_lens"])
            cap = max(s["kv_lens"]) + 13
            s["q"] = normal(rows, H, D)
            cache = normal(2, len(lens) * cap, K, D)
            s["k"], s["v"] = cache[0], cache[1]
            s["kv_starts"] = [i * cap for i in range(len(lens))]
        else:
            s["kv_lens"] = lens
            qkv = normal(rows, H + 2 * K, D)
            s["q"], s["k"], s["v"] = qkv[:, :H], qkv[:, H:H + K], qkv[:, H + K:]
            s["kv_starts"] = list(np.cumsum([0] + lens[:-1]))
        starts = np.cumsum([0] + lens)
        s["d_q_start"] = torch.tensor(starts, dtype=torch.int32).cuda()
        s["d_kv_start"] = torch.tensor(np.array(s["kv_starts"]), dtype=torch.int64).cuda()
        s["d_kv_len"] = torch.tensor(s["kv_lens"], dtype=torch.int32).cuda()
    if own:
        s["call"] = _handle(case, s, dt)
    return s


# ---- plain forms -----------------------------------------------------------

def _frequencies(case):
    """Radians a position of each pair, in 64 bits, and the factor of cosine and sine."""
    r = case["rotary"]
    f = case["theta"] ** (-torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r)
    if case["scaling"] == "linear":
        return f / 4.0, 1.0
    if case["scaling"] == "yarn":  # factor 16 over 16384 positions, turns 32 and 1
        edge = [r * math.log(16384.0 / (t * 2 * math.pi)) / (2 * math.log(case["theta"])) for t in (32.0, 1.0)]
        lo, hi = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), r - 1)
        ramp = ((torch.arange(r // 2, dtype=torch.float64, device="cuda") - lo) / max(0.001, hi - lo)).clamp(0, 1)
        return f / 16.0 * ramp + f * (1 - ramp), 0.1 * math.log(16.0) + 1
    if case["scaling"] == "bands":  # factor 8 over 8192 positions, bands 1 and 4
        smooth = ((8192.0 * f / (2 * math.pi) - 1.0) / 3.0).clamp(0, 1)
        return (1 - smooth) * f / 8.0 + smooth * f, 1.0
    return f, 1.0


def _plain_rope(case, s):
    f, m = _frequencies(case)
    angle = s["positions"].double()[:, None] * f
    c, sn = (m * angle.cos()).float()[:, None], (m * angle.sin()).float()[:, None]
    r = case["rotary"]

    def turn(x):
        y = x.float().clone()
        if case["layout"] == "half":
            a, b = y[..., :r // 2].clone(), y[..., r // 2:r].clone()
            y[..., :r // 2], y[..., r // 2:r] = a * c - b * sn, a * sn + b * c
        else:
            a, b = y[..., 0:r:2].clone(), y[..., 1:r:2].clone()
            y[..., 0:r:2], y[..., 1:r:2] = a * c - b * sn, a * sn + b * c
        return y.to(x.dtype)

    return turn(s["q"]), turn(s["k"])


def _plain_norm(case, s):
    h = s["x"].float() + s["delta"].float()
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS) * s["w"]
    group = case["group"] or case["hidden"]
    blocks = y.view(case["rows"], -1, group)
    top = 127.0 if case["type8"] == "i8" else 448.0
    scale = blocks.abs().amax(-1, keepdim=True) / top
    q = blocks / torch.where(scale > 0, scale, torch.ones_like(scale))
    # bytes as the values they stand for; 8-bit floats are that in units of their scale
    q = (q.round() * scale).half() if case["type8"] == "i8" else q.clamp(-top, top).to(torch.float8_e4m3fn)
    out = [h.to(s["x"].dtype), q.view(case["rows"], -1), scale.squeeze(-1)]
    return out + [y.to(s["x"].dtype)] if case["both"] else out


def _plain_attention(case, s):
    """Blocks of CHUNK queries of one request, each against the keys of its
    window and the first keys, gathered; one product over all blocks."""
    H, K, D = case["heads"], case["kv_heads"], case["head_dim"]
    left, right, sinks = case["left"], case["right"], case["sinks"]
    n, m = torch.tensor(s["q_lens"]), torch.tensor(s["kv_lens"])
    chunk, most = min(CHUNK, int(n.max())), max(1, int(m.max()))
    parts = (n + chunk - 1) // chunk
    b = torch.repeat_interleave(torch.arange(len(n)), parts)
    first = (torch.arange(len(b)) - torch.repeat_interleave(parts.cumsum(0) - parts, parts)) * chunk
    row0 = (n.cumsum(0) - n)[b]
    at = first[:, None] + torch.arange(chunk)  # query of its request
    real = at < n[b][:, None]
    p = at + (m - n)[b][:, None]
    span = left + chunk + right if left >= 0 and right >= 0 else most
    start = (p[:, 0] - left).clamp(min=0) if left >= 0 else torch.zeros_like(first)
    if span >= most:
        span, start = most, torch.zeros_like(first)
    j = torch.cat([torch.arange(sinks if left >= 0 else 0).expand(len(b), -1), start[:, None] + torch.arange(span)], 1)
    extra = torch.arange(j.shape[1]) < j.shape[1] - span
    p, j, real, b, m, at, row0, extra = (t.cuda() for t in (p, j, real, b, m, at, row0, extra))
    low = p[:, :, None] - left if left >= 0 else torch.zeros_like(p)[:, :, None]
    jj = j[:, None, :]
    end = torch.minimum(m[b][:, None, None], p[:, :, None] + right + 1) if right >= 0 else m[b][:, None, None]
    start = start.cuda()[:, None, None]
    seen = (jj < end) & torch.where(extra, jj < torch.minimum(low, start), (jj >= low) | (jj < sinks))
    rows = (row0[:, None] + at).clamp(max=s["q"].shape[0] - 1)
    kv = (s["d_kv_start"][b][:, None] + torch.minimum(j, (m[b][:, None] - 1).clamp(min=0))).clamp(
        max=s["k"].shape[0] - 1)
    q = s["q"][rows].float().view(len(b), chunk, K, H // K, D).permute(0, 2, 1, 3, 4).reshape(len(b), K, -1, D)
    keys = s["k"][kv].float().permute(0, 2, 3, 1).contiguous()
    values = s["v"][kv].float().permute(0, 2, 1, 3).contiguous()
    scores = (q @ keys).view(len(b), K, chunk, H // K, -1) * D ** -0.5
    scores = scores.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = scores.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = e.sum(-1, keepdim=True)
    o = (e.view(len(b), K, chunk * (H // K), -1) @ values).view(len(b), K, chunk, H // K, D)
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    o = o.permute(0, 2, 1, 3, 4).reshape(len(b), chunk, H, D)
    return o[real].to(s["q"].dtype)


# ---- the package's kernels --------------------------------------------------

def _handle(case, s, dt):
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from nemo_amd import operators as ops
    code = {"f16": ops.TYPE_F16, "bf16": ops.TYPE_BF16, "f32": ops.TYPE_F32}[case["type"]]
    if case["op"] == "rope":
        rope = ops.Rope(ops.rope_config(
            case["head_dim"], rotary_dim=case["rotary"], theta=case["theta"],
            layout={"interleaved": ops.ROPE_INTERLEAVED, "half": ops.ROPE_HALF}[case["layout"]],
            **{"none": {}, "linear": dict(scaling=ops.ROPE_LINEAR, factor=4.0),
               "yarn": dict(scaling=ops.ROPE_YARN, factor=16.0, original_positions=16384),
               "bands": dict(scaling=ops.ROPE_BANDS, factor=8.0, original_positions=8192, low_band=1.0,
                             high_band=4.0)}[case["scaling"]]))
        s["out"] = (torch.empty_like(s["q"]), torch.empty_like(s["k"]))
        heads = [ops.rope_heads(x.data_ptr(), y.data_ptr(), x.shape[1], case["head_dim"])
                 for x, y in zip((s["q"], s["k"]), s["out"])]
        rows, positions = case["rows"], s["positions"].data_ptr()

        def call():
            rope.apply(code, heads[0], heads[1], rows, positions, stream=torch.cuda.current_stream().cuda_stream)
            return s["out"]
        return call
    if case["op"] == "norm":
        rows, hidden = case["rows"], case["hidden"]
        blocks = hidden // case["group"] if case["group"] else 1
        i8 = case["type8"] == "i8"
        h, y = torch.empty_like(s["x"]), torch.empty_like(s["x"]) if case["both"] else None
        y8 = torch.empty(rows, hidden, dtype=torch.int8 if i8 else torch.float8_e4m3fn, device="cuda")
        scales = torch.empty(rows, blocks, dtype=torch.float32, device="cuda")
        args = ops.norm_args(code, rows, hidden, s["x"].data_ptr(), s["w"].data_ptr(), EPS,
                             d_delta=s["delta"].data_ptr(), d_sum=h.data_ptr(), d_y=y.data_ptr() if case["both"] else 0,
                             d_y8=y8.data_ptr(), type8=ops.TYPE_I8 if i8 else ops.TYPE_E4M3, d_scales=scales.data_ptr(),
                             group=case["group"])
        norm = ops.RmsNorm()
        values = torch.empty(rows, hidden, dtype=torch.float16, device="cuda") if i8 else y8
        out = [h, values, scales, y] if case["both"] else [h, values, scales]

        def call():
            norm.run(args, stream=torch.cuda.current_stream().cuda_stream)
            if i8:  # the values that the bytes stand for
                torch.mul(y8.view(rows, blocks, -1), scales[..., None], out=values.view(rows, blocks, -1))
            return out
        return call
    H, K, D = case["heads"], case["kv_heads"], case["head_dim"]
    attention = ops.WindowAttention(ops.attention_config(H, K, D, code, left=case["left"], right=case["right"],
                                                         sinks=case["sinks"]))
    out = torch.empty(s["q"].shape[0], H, D, dtype=dt, device="cuda")
    need = attention.workspace_bytes(len(s["q_lens"]), s["q"].shape[0], max(s["kv_lens"]))
    s["workspace"] = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    batch = ops.attention_batch(
        len(s["q_lens"]), s["q"].shape[0], s["k"].shape[0], max(s["kv_lens"]), s["d_q_start"].data_ptr(),
        s["d_kv_start"].data_ptr(), s["d_kv_len"].data_ptr(),
        *((t.data_ptr(), t.stride(0), t.stride(1)) for t in (s["q"], s["k"], s["v"], out)),
        d_workspace=s["workspace"].data_ptr(), workspace_bytes=need)

    def call():
        attention.run(batch, stream=torch.cuda.current_stream().cuda_stream)
        return out
    return call


def run(state):
    if own:
        return state["call"]()
    return {"rope": _plain_rope, "norm": _plain_norm, "attention": _plain_attention}[state["case"]["op"]](
        state["case"], state)


# ---- what a pass cannot do without ------------------------------------------

def _windows(case):
    """Of each request: first and past-last window key of every query, and the sinks outside it."""
    n, m = _ints(case["q_lens"]), _ints(case["kv_lens"] or case["q_lens"])
    for a, b in zip(n, m):
        p = np.arange(a, dtype=np.int64) + b - a
        hi = np.clip(p + case["right"] + 1, 0, b) if case["right"] >= 0 else np.full(a, b, dtype=np.int64)
        lo = np.clip(p - case["left"], 0, hi) if case["left"] >= 0 else np.zeros(a, dtype=np.int64)
        yield lo, hi, np.minimum(np.minimum(case["sinks"], lo), hi)


def work(case):
    size = SIZE[case["type"]]
    if case["op"] == "rope":
        heads = case["heads"] + case["kv_heads"]
        return {"bytes": 2 * size * case["rows"] * heads * case["head_dim"] + 8 * case["rows"],
                "flops": 3 * case["rows"] * heads * case["rotary"]}
    if case["op"] == "norm":
        values = case["rows"] * case["hidden"]
        blocks = case["rows"] * (case["hidden"] // case["group"] if case["group"] else 1)
        return {"bytes": values * (size * (4 if case["both"] else 3) + 1) + 4 * blocks + 4 * case["hidden"],
                "flops": 8 * values}
    H, K, D = case["heads"], case["kv_heads"], case["head_dim"]
    seen, keys, rows = 0, 0, 0
    for lo, hi, sinks in _windows(case):
        seen += int((hi - lo + sinks).sum())
        keys += int(hi.max() - lo.min()) + int(min(case["sinks"], lo.min()))
        rows += len(lo)
    return {"bytes": size * D * (2 * rows * H + 2 * keys * K), "flops": 4 * D * H * seen}


# ---- 64 bits ----------------------------------------------------------------

def exact(case, seed):
    """The operators from their definitions in 64 bits."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"rope": _exact_rope, "norm": _exact_norm, "attention": _exact_attention}[case["op"]](case, s)


def _exact_rope(case, s):
    r = case["rotary"]
    turns = []
    for i in range(r // 2):
        f = math.exp(-2.0 * i / r * math.log(case["theta"]))
        wave = 2 * math.pi / f
        if case["scaling"] == "linear":
            f = f / 4
        elif case["scaling"] == "yarn":
            pair = [r * math.log(16384 / (2 * math.pi * t)) / (2 * math.log(case["theta"])) for t in (32, 1)]
            lo, hi = max(0, math.floor(pair[0])), min(r - 1, math.ceil(pair[1]))
            keep = 1 - min(1.0, max(0.0, (i - lo) / max(0.001, hi - lo)))
            f = f * (keep + (1 - keep) / 16)
        elif case["scaling"] == "bands":
            if wave > 8192 / 1.0:
                f = f / 8
            elif wave > 8192 / 4.0:
                keep = (8192 / wave - 1) / (4 - 1)
                f = f * (keep + (1 - keep) / 8)
        turns.append(f)
    angle = s["positions"].double()[:, None, None] * torch.tensor(turns, dtype=torch.float64, device="cuda")
    m = 1 + 0.1 * math.log(16) if case["scaling"] == "yarn" else 1.0
    by = torch.polar(torch.full_like(angle, m), angle)

    def turn(x):
        x = x.double()
        part = x[..., :r]
        if case["layout"] == "half":
            z = torch.complex(part[..., :r // 2].contiguous(), part[..., r // 2:].contiguous()) * by
            part = torch.cat([z.real, z.imag], -1)
        else:
            z = torch.view_as_complex(part.reshape(*part.shape[:-1], r // 2, 2).contiguous()) * by
            part = torch.view_as_real(z).flatten(-2)
        return torch.cat([part, x[..., r:]], -1)

    return turn(s["q"]), turn(s["k"])


def _exact_norm(case, s):
    h = s["x"].double().add(s["delta"].double())
    y = h * torch.rsqrt(torch.linalg.vector_norm(h, dim=-1, keepdim=True) ** 2 / case["hidden"] + EPS)
    y = y * s["w"].double()
    parts = y.unflatten(-1, (-1, case["group"] or case["hidden"]))
    peak = torch.maximum(parts.amax(-1), -parts.amin(-1))
    if case["type8"] == "i8":
        step = peak[..., None] / 127
        values = torch.round(parts / step) * step
    else:
        # 3 bits behind the leading one, down to 2^-9 in units of the scale
        unit = parts * 448 / peak[..., None]
        e = torch.floor(torch.log2(unit.abs().clamp(min=2.0 ** -20))).clamp(min=-6)
        values = torch.round(unit * 2.0 ** (3 - e)) * 2.0 ** (e - 3)
    out = [h, values.flatten(-2), peak / (127 if case["type8"] == "i8" else 448)]
    return out + [y] if case["both"] else out


def _exact_attention(case, s):
    H, K, D = case["heads"], case["kv_heads"], case["head_dim"]
    out = torch.zeros(sum(s["q_lens"]), H, D, dtype=torch.float64, device="cuda")
    row = 0
    for (lo, hi, sinks), start in zip(_windows(case), s["kv_starts"]):
        for at in range(0, len(lo), 512):
            part = slice(at, min(at + 512, len(lo)))
            # the block's keys: from its lowest window key on, behind the sinks that lie before that
            first, last = int(lo[part].min()), int(hi[part].max())
            pick = np.concatenate([np.arange(min(case["sinks"], first)), np.arange(first, last)])
            if len(pick):
                j = torch.from_numpy(pick).cuda()
                a, b = (torch.from_numpy(t[part])[:, None].cuda() for t in (lo, hi))
                hidden = (j >= b) | ((j < a) & (j >= case["sinks"]))
                q = s["q"][row + at:row + at + hidden.shape[0]].double().transpose(0, 1)
                for g in range(K):
                    k = s["k"][start + j, g].double()
                    v = s["v"][start + j, g].double()
                    t = q[g * (H // K):(g + 1) * (H // K)] @ k.t().contiguous() / math.sqrt(D)
                    t = torch.softmax(t.masked_fill(hidden, -math.inf), -1)
                    t = torch.nan_to_num(t, nan=0.0)
                    out[row + at:row + at + hidden.shape[0], g * (H // K):(g + 1) * (H // K)] = (t @ v).transpose(0, 1)
        row += len(lo)
    return out
