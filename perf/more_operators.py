"""What the speed of the low-bit operators of an attention block is measured
on: norms of query and key heads with their rotation, products of 8-bit rows,
appending keys and values to a paged cache of 4-bit floats, and attention over
that cache, each in a plain form of elementary torch operations and through
the package's kernels, with inputs made from a seed alone and 64-bit results.

Heads, keys and values are N(0, 1), norm weights N(1, 0.1); 8-bit rows and
weights are N(0, 1) rounded to steps of max / 127, as a row's quantization
leaves them; caches hold N(0, 1) in 4 bits, their pages in random order.

A page of a cache (tokens of all KV heads, head by head) holds P tokens of D
values of K and of V: K's codes [P][D / 2], V's codes [P / 4][16][4][D / 32]
(16 pieces of D / 16 values), scales of K and of V [P / 8][D / 32][8]. Codes
are E2M1 floats, two a byte, the first in the low bits; scales are powers of
two, 2^(byte - 127), of 32 values of a head.
"""
import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PACKAGE = os.path.join(_ROOT, "nemotron-3-embed-webgpu_amd")

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
EPS = 1e-5
CHUNK = 256  # queries of a block of the plain attention
MAGNITUDES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _heads(name, type_, rows, heads, kv_heads, head_dim, rotary, layout, theta):
    c = {"op": "heads", "type": type_, "rows": rows, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
         "rotary": rotary, "layout": layout, "theta": theta}
    return dict(c, name=name) if name else c


def _matmul(name, type_, m, n, k, bias):
    c = {"op": "matmul", "type": type_, "m": m, "n": n, "k": k, "bias": bias}
    return dict(c, name=name) if name else c


def _append(name, type_, kv_heads, head_dim, page, layout, q_lens, kv_lens):
    c = {"op": "append", "type": type_, "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "layout": layout,
         "q_lens": ",".join(map(str, q_lens)), "kv_lens": ",".join(map(str, kv_lens))}
    return dict(c, name=name) if name else c


def _attention(name, type_, heads, kv_heads, head_dim, page, left, sinks, q_lens, kv_lens):
    c = {"op": "attention", "type": type_, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
         "left": left, "sinks": sinks, "q_lens": ",".join(map(str, q_lens)), "kv_lens": ",".join(map(str, kv_lens))}
    return dict(c, name=name) if name else c


# how far 64 conversations have come
CACHED = [97 + (i * i * 7919 + 613 * i) % 32600 for i in range(64)]


def listed():
    return [
        # one token's query and key heads, as each step of a decoder norms and turns them
        _heads("heads_1_token", "f16", 1, 32, 8, 128, 128, "half", 1e6),
        # a long document's heads, of which a part is turned
        _heads("heads_16001", "bf16", 16001, 32, 8, 128, 96, "interleaved", 5e5),
        # one token through a fused projection of queries, keys and values
        _matmul("matmul_1x5120x2048", "f16", 1, 5120, 2048, False),
        # the next token of 77 conversations, down projection with a bias
        _matmul("matmul_77x2048x6144", "bf16", 77, 2048, 6144, True),
        # a benchmark batch of 16 passages through gate and up
        _matmul("matmul_2400x12288x2048", "f16", 2400, 12288, 2048, False),
        # a long document through a wide layer
        _matmul("matmul_16384x8192x8192", "bf16", 16384, 8192, 8192, False),
        # the next token of 64 conversations goes into their caches
        _append("append_64_tokens", "bf16", 8, 128, 64, "half", [1] * 64, CACHED),
        # prompts of all lengths, some behind what is cached
        _append("append_prompts", "f16", 8, 128, 32, "interleaved", [20000, 1, 5003, 777, 64, 6001],
                [20000, 4097, 5003, 9000, 64, 70001]),
        # one conversation's next token: the smallest attention
        _attention("attention_1_token", "f16", 32, 8, 64, 32, 1023, 4, [1], [5000]),
        # the next token of 64 conversations of all lengths
        _attention("attention_64_tokens", "bf16", 32, 8, 128, 64, -1, 0, [1] * 64, CACHED),
        # the next token of one long document, every key visible
        _attention("attention_1_token_all", "f16", 32, 8, 128, 128, -1, 0, [1], [131072]),
        # prompts arriving in pieces behind what is cached
        _attention("attention_pieces", "bf16", 32, 8, 128, 64, -1, 0, [2048, 77, 1, 300], [18001, 77, 4097, 1300]),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["heads", "matmul", "matmul", "append", "attention", "attention"])
    if op == "heads":
        head_dim = rng.choice([64, 64, 80, 96, 128, 128, 256])
        rotary = head_dim if rng.random() < 0.6 else 2 * rng.randint(4, head_dim // 2)
        kv_heads = rng.choice([1, 2, 3, 8])
        return _heads("", rng.choice(["f16", "bf16", "f32"]), _log_int(rng, 1, 4096), kv_heads * rng.choice([1, 3, 4]),
                      kv_heads, head_dim, rotary, rng.choice(["interleaved", "half"]), rng.choice([1e4, 5e5, 1e6]))
    if op == "matmul":
        return _matmul("", rng.choice(["f16", "bf16", "f32"]), _log_int(rng, 1, 8192), _log_int(rng, 64, 8192),
                       _log_int(rng, 64, 8192), rng.random() < 0.5)
    head_dim, type_ = rng.choice([64, 128]), rng.choice(["f16", "bf16"])
    kv_heads, page = rng.choice([1, 2, 4, 8]), rng.choice([32, 64, 128, 256])
    count = rng.randint(1, 8)
    one = rng.random() < 0.5
    if op == "append":
        lens = [1 if one else _log_int(rng, 1, 3000) for _ in range(count)]
        return _append("", rng.choice(["f16", "bf16", "f32"]), rng.choice([kv_heads, 3]), head_dim, page,
                       rng.choice(["interleaved", "half"]), lens, [n + _log_int(rng, 1, 9000) - 1 for n in lens])
    heads = kv_heads * min(rng.choice([1, 2, 3, 4, 5, 8]), 32 // kv_heads)
    lens = [1 if one else _log_int(rng, 1, 300) for _ in range(count)]
    return _attention("", type_, heads, kv_heads, head_dim, page, rng.choice([-1, -1, _log_int(rng, 64, 4096)]),
                      rng.choice([0, 0, 4, 100]), lens, [n + _log_int(rng, 1, 32000 if one else 9000) - 1 for n in lens])


def _ints(text):
    return [int(t) for t in text.split(",")]


# ---- inputs -----------------------------------------------------------------

def _rows8(g, rows, k):
    """8-bit rows with their scales, as a row's quantization leaves them; rows begin on 16 bytes."""
    codes = torch.empty(rows, (k + 15) // 16 * 16, dtype=torch.int8, device="cuda")
    scales = torch.empty(rows, dtype=torch.float32, device="cuda")
    for at in range(0, rows, 4096):
        x = torch.randn(min(4096, rows - at), codes.shape[1], generator=g, device="cuda", dtype=torch.float32)
        s = x[:, :k].abs().amax(-1, keepdim=True) / 127
        codes[at:at + x.shape[0]] = (x / s).round().clamp(-127, 127).to(torch.int8)
        scales[at:at + x.shape[0]] = s.squeeze(-1)
    return codes, scales


def _codes4(x):
    """Codes and scale bytes of float32 values [..., D]."""
    blocks = x.unflatten(-1, (-1, 32))
    part, power = torch.frexp(blocks.abs().amax(-1, keepdim=True))
    s = power - 3 + (part > 0.875).int()
    unit = (blocks * torch.exp2(-s.float())).flatten(-2)
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=x.device)
    codes = torch.bucketize(unit.abs(), borders, out_int32=True).to(torch.uint8) | ((unit < 0).to(torch.uint8) << 3)
    return codes, (s.squeeze(-1) + 127).to(torch.uint8)


def _page_bytes(case):
    return case["kv_heads"] * case["page"] * (case["head_dim"] + case["head_dim"] // 16)


def _pages(case, g, pages):
    """Pages of N(0, 1) keys and values."""
    H, D, P = case["kv_heads"], case["head_dim"], case["page"]
    data = torch.empty(pages, _page_bytes(case), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // (P * H * D))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        parts = []
        for values in (False, True):
            codes, scales = _codes4(torch.randn(n, P, H, D, generator=g, device="cuda"))
            two = (codes[..., 0::2] | (codes[..., 1::2] << 4)).permute(0, 2, 1, 3)  # [n, H, P, D / 2]
            if values:
                two = two.reshape(n, H, P // 4, 4, 16, D // 32).transpose(3, 4)
            scales = scales.reshape(n, P // 8, 8, H, D // 32).permute(0, 3, 1, 4, 2)
            parts.append((two.reshape(n, H, -1), scales.reshape(n, H, -1)))
        (k, ks), (v, vs) = parts
        data[at:at + n] = torch.cat([k, v, ks, vs], -1).reshape(n, -1)
    return data


def _table(case, g, kv_lens):
    """Pages of each request, in random order, and how many there are."""
    per = [(n + case["page"] - 1) // case["page"] for n in kv_lens]
    order = torch.randperm(sum(per), generator=g, device="cuda").int()
    table = torch.zeros(len(per), max(per), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    return table, at


def prepare(case, seed):
    """Inputs on the GPU, outputs' buffers and, for the package's kernels, the handle that a program keeps."""
    g = torch.Generator(device="cuda")
    g.manual_seed(1 + int(seed))
    dt = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    s = {"case": case}
    if case["op"] == "heads":
        rows, d = case["rows"], case["head_dim"]
        s["q"], s["k"] = normal(rows, case["heads"], d).to(dt), normal(rows, case["kv_heads"], d).to(dt)
        s["q_weight"], s["k_weight"] = 1 + 0.1 * normal(d), 1 + 0.1 * normal(d)
        s["positions"] = torch.arange(rows, dtype=torch.int64, device="cuda") + 1000 + int(seed) % 7
    elif case["op"] == "matmul":
        s["x"], s["x_scale"] = _rows8(g, case["m"], case["k"])
        s["w"], s["w_scale"] = _rows8(g, case["n"], case["k"])
        s["bias"] = normal(case["n"]) if case["bias"] else None
    else:
        q_lens, kv_lens = _ints(case["q_lens"]), _ints(case["kv_lens"])
        s["q_lens"], s["kv_lens"] = q_lens, kv_lens
        K, D, rows = case["kv_heads"], case["head_dim"], sum(q_lens)
        s["table"], s["pages"] = _table(case, g, kv_lens)
        starts = [0]
        for n in q_lens:
            starts.append(starts[-1] + n)
        s["q_start"] = torch.tensor(starts, dtype=torch.int32).cuda()
        s["kv_len"] = torch.tensor(kv_lens, dtype=torch.int32).cuda()
        if case["op"] == "append":
            kv = normal(rows, 2 * K, D).to(dt)  # as a projection leaves them
            s["k"], s["v"] = kv[:, :K], kv[:, K:]
            s["data"] = torch.zeros(s["pages"], _page_bytes(case), dtype=torch.uint8, device="cuda")
        else:
            s["q"] = normal(rows, case["heads"], D).to(dt)
            s["data"] = _pages(case, g, s["pages"])
    if own:
        s["call"] = _handle(case, s, dt)
    return s


# ---- plain forms ------------------------------------------------------------

def _turn(x, c, s, r, half):
    """Pairs of the last axis's first r values turned; x is changed."""
    first, second = (slice(0, r // 2), slice(r // 2, r)) if half else (slice(0, r, 2), slice(1, r, 2))
    a, b = x[..., first].clone(), x[..., second].clone()
    x[..., first], x[..., second] = a * c - b * s, a * s + b * c
    return x


def _plain_heads(case, s):
    r = case["rotary"]
    f = case["theta"] ** (-torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r)
    angle = s["positions"].double()[:, None, None] * f
    c, sn = angle.cos().float(), angle.sin().float()

    def one(x, w):
        x = x.float()
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        return _turn(x, c, sn, r, case["layout"] == "half")

    dt = s["q"].dtype
    return one(s["q"], s["q_weight"]).to(dt), one(s["k"], s["k_weight"]).to(dt)


def _plain_matmul(case, s):
    k = case["k"]
    y = s["x"][:, :k].float() @ s["w"][:, :k].float().t()
    y = y * s["x_scale"][:, None] * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(TYPES[case["type"]])


def _power(s):
    """2^s of integers, in 64 bits."""
    return ((s.long() + 1023) << 52).view(torch.float64)


def _plain_append(case, s):
    """In 64 bits: a value next to a border of two codes would fall on either side."""
    D = case["head_dim"]
    n, m = torch.tensor(s["q_lens"]), torch.tensor(s["kv_lens"])
    at = torch.arange(int(n.sum())) - torch.repeat_interleave(n.cumsum(0) - m, n)  # each row's token of its request
    f = 1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
    angle = at.cuda().double()[:, None, None] * f
    k = _turn(s["k"].double(), angle.cos(), angle.sin(), D, case["layout"] == "half")
    table = torch.tensor(MAGNITUDES, dtype=torch.float64, device="cuda")

    def held(x):
        blocks = x.unflatten(-1, (-1, 32))
        part, power = torch.frexp(blocks.abs().amax(-1, keepdim=True))
        scale = _power(power - 3 + (part > 0.875).int())
        unit = blocks / scale
        a = unit.abs()
        code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int()
                + (a >= 3.5).int() + (a > 5.0).int())
        return (torch.copysign(table[code], unit) * scale).flatten(-2).half()

    return held(k), held(s["v"].double())


def _plain_attention(case, s):
    """Caches decoded request by request; blocks of CHUNK queries of one
    request against all of its keys, one product over all blocks."""
    H, K, D, P = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    pages = s["data"][s["table"].long()]  # [count, pages, bytes of a page]
    count, per = pages.shape[:2]
    k, v, ks, vs = pages.view(count, per, K, -1).split([P * D // 2, P * D // 2, P * D // 32, P * D // 32], -1)
    table = torch.tensor(MAGNITUDES + [-x for x in MAGNITUDES], device="cuda")

    def decoded(codes, scales):  # codes [count, per, K, P, D / 2] -> [count, keys, K, D]
        x = table[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()]
        scales = scales.reshape(count, per, K, P // 8, D // 32, 8).transpose(4, 5).reshape(count, per, K, P, D // 32)
        x = x.unflatten(-1, (-1, 32)) * torch.exp2(scales.float() - 127)[..., None]
        return x.flatten(-2).transpose(2, 3).reshape(count, per * P, K, D)

    k = decoded(k.reshape(count, per, K, P, D // 2), ks)
    v = decoded(v.reshape(count, per, K, P // 4, 16, 4, D // 32).transpose(4, 5).reshape(count, per, K, P, D // 2), vs)
    n, m = torch.tensor(s["q_lens"]), torch.tensor(s["kv_lens"])
    chunk = min(CHUNK, int(n.max()))
    parts = (n + chunk - 1) // chunk
    b = torch.repeat_interleave(torch.arange(len(n)), parts)
    first = (torch.arange(len(b)) - torch.repeat_interleave(parts.cumsum(0) - parts, parts)) * chunk
    at = first[:, None] + torch.arange(chunk)  # query of its request
    real = (at < n[b][:, None]).cuda()
    p = (at + (m - n)[b][:, None]).cuda()[:, :, None]
    rows = ((n.cumsum(0) - n)[b][:, None] + at).clamp(max=s["q"].shape[0] - 1).cuda()
    j = torch.arange(per * P, device="cuda")
    seen = j <= p
    if case["left"] >= 0:
        seen &= (j >= p - case["left"]) | (j < case["sinks"])
    b = b.cuda()
    q = s["q"][rows].float().view(len(b), chunk, K, H // K, D).permute(0, 2, 1, 3, 4).reshape(len(b), K, -1, D)
    scores = (q @ k[b].permute(0, 2, 3, 1)).view(len(b), K, chunk, H // K, -1) * D ** -0.5
    scores = scores.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    e = scores.sub_(scores.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = e.sum(-1, keepdim=True)
    o = (e.view(len(b), K, chunk * (H // K), -1) @ v[b].transpose(1, 2)).view(len(b), K, chunk, H // K, D) / total
    return o.permute(0, 2, 1, 3, 4).reshape(len(b), chunk, H, D)[real].to(s["q"].dtype)


# ---- the package's kernels ----------------------------------------------------

def _handle(case, s, dt):
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from nemo_amd import operators as ops
    code = {"f16": ops.TYPE_F16, "bf16": ops.TYPE_BF16, "f32": ops.TYPE_F32}[case["type"]]
    layout = {"interleaved": ops.ROPE_INTERLEAVED, "half": ops.ROPE_HALF}[case.get("layout", "half")]

    def stream():
        return torch.cuda.current_stream().cuda_stream

    if case["op"] == "heads":
        rope = ops.Rope(ops.rope_config(case["head_dim"], rotary_dim=case["rotary"], theta=case["theta"], layout=layout))
        out = (torch.empty_like(s["q"]), torch.empty_like(s["k"]))
        heads = [ops.rope_heads(x.data_ptr(), y.data_ptr(), x.shape[1], case["head_dim"])
                 for x, y in zip((s["q"], s["k"]), out)]
        norm = ops.head_norm(s["q_weight"].data_ptr(), s["k_weight"].data_ptr(), EPS)
        rows, positions = case["rows"], s["positions"].data_ptr()

        def call():
            rope.norm_apply(code, heads[0], heads[1], norm, rows, positions, stream=stream())
            return out
        return call
    if case["op"] == "matmul":
        y = torch.empty(case["m"], case["n"], dtype=dt, device="cuda")
        args = ops.matmul8_args(code, case["m"], case["n"], case["k"], s["x"].data_ptr(), s["x_scale"].data_ptr(),
                                s["w"].data_ptr(), s["w_scale"].data_ptr(), y.data_ptr(),
                                d_bias=s["bias"].data_ptr() if case["bias"] else 0, x_row=s["x"].stride(0),
                                w_row=s["w"].stride(0))
        matmul = ops.Matmul8()

        def call():
            matmul.run(args, stream=stream())
            return y
        return call
    K, D = case["kv_heads"], case["head_dim"]
    cache = ops.Cache4(ops.cache4_config(K, D, case["page"]))
    pages = ops.cache4_pages(len(s["q_lens"]), s["pages"], s["data"].data_ptr(), s["table"].data_ptr(),
                             s["table"].shape[1], s["kv_len"].data_ptr())
    rows = sum(s["q_lens"])
    if case["op"] == "append":
        rope = ops.Rope(ops.rope_config(D, theta=1e6, layout=layout))
        out = torch.empty(2, rows, K, D, dtype=torch.float16, device="cuda")
        new, held = (ops.cache4_rows(t, rows, s["q_start"].data_ptr(), *((x.data_ptr(), x.stride(0), x.stride(1))
                                                                         for x in kv))
                     for t, kv in ((code, (s["k"], s["v"])), (ops.TYPE_F16, (out[0], out[1]))))

        def call():
            cache.append(pages, new, rope, stream=stream())
            cache.read(pages, held, stream=stream())  # the values that the codes stand for
            return out[0], out[1]
        return call
    config = ops.attention_config(case["heads"], K, D, code, left=case["left"], right=0, sinks=case["sinks"])
    out = torch.empty_like(s["q"])
    need = cache.workspace_bytes(config, len(s["q_lens"]), rows, max(s["kv_lens"]))
    s["workspace"] = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    queries = ops.cache4_queries(rows, max(s["kv_lens"]), s["q_start"].data_ptr(),
                                 *((t.data_ptr(), t.stride(0), t.stride(1)) for t in (s["q"], out)),
                                 d_workspace=s["workspace"].data_ptr(), workspace_bytes=need)

    def call():
        cache.attention(config, pages, queries, stream=stream())
        return out
    return call


def run(state):
    if own:
        return state["call"]()
    return {"heads": _plain_heads, "matmul": _plain_matmul, "append": _plain_append, "attention": _plain_attention}[
        state["case"]["op"]](state["case"], state)


# ---- what a pass cannot do without ----------------------------------------------

def _windows(case):
    """Of each request's queries: first and past-last key of the window, and the sinks before it."""
    for n, m in zip(_ints(case["q_lens"]), _ints(case["kv_lens"])):
        hi = torch.arange(n) + m - n + 1
        lo = (hi - 1 - case["left"]).clamp(min=0) if case["left"] >= 0 else torch.zeros_like(hi)
        yield lo, hi, lo.clamp(max=case["sinks"])


def work(case):
    size = SIZE[case["type"]]
    if case["op"] == "heads":
        values = case["rows"] * (case["heads"] + case["kv_heads"]) * case["head_dim"]
        return {"bytes": 2 * size * values + 8 * case["rows"] + 8 * case["head_dim"], "flops": 7 * values}
    if case["op"] == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + size * m * n + 4 * (m + n) + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    K, D = case["kv_heads"], case["head_dim"]
    if case["op"] == "append":  # rows read, codes and scales written, and read again as values of 16 bits
        values = 2 * K * D * sum(_ints(case["q_lens"]))
        return {"bytes": values * (size + 2 * (0.5 + 1 / 32) + 2), "flops": 10 * values}
    H, seen, keys, rows = case["heads"], 0, 0, 0
    for lo, hi, sinks in _windows(case):
        seen += int((hi - lo + sinks).sum())
        keys += int(hi.max() - lo.min()) + int(sinks.min())
        rows += len(lo)
    return {"bytes": 2 * SIZE[case["type"]] * rows * H * D + keys * K * (D + D // 16), "flops": 4 * D * H * seen}


# ---- 64 bits -----------------------------------------------------------------------

def exact(case, seed):
    """The operators from their definitions in 64 bits."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"heads": _exact_heads, "matmul": _exact_matmul, "append": _exact_append, "attention": _exact_attention}[
        case["op"]](case, s)


def _exact_turn(x, positions, r, theta, half):
    turns = torch.tensor([math.exp(-2.0 * i / r * math.log(theta)) for i in range(r // 2)], dtype=torch.float64,
                         device="cuda")
    angle = positions.double()[:, None, None] * turns
    by = torch.polar(torch.ones_like(angle), angle)
    part = x[..., :r]
    if half:
        z = torch.complex(part[..., :r // 2].contiguous(), part[..., r // 2:].contiguous()) * by
        part = torch.cat([z.real, z.imag], -1)
    else:
        z = torch.view_as_complex(part.reshape(*part.shape[:-1], r // 2, 2).contiguous()) * by
        part = torch.view_as_real(z).flatten(-2)
    return torch.cat([part, x[..., r:]], -1)


def _exact_heads(case, s):
    out = []
    for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        x = x.double()
        x = x * torch.rsqrt(torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / x.shape[-1] + EPS) * w.double()
        out.append(_exact_turn(x, s["positions"], case["rotary"], case["theta"], case["layout"] == "half"))
    return out[0], out[1]


def _exact_matmul(case, s):
    k, parts = case["k"], []
    w = s["w"][:, :k].double() * s["w_scale"].double()[:, None]
    for at in range(0, case["m"], 4096):
        x = s["x"][at:at + 4096, :k].double() * s["x_scale"][at:at + 4096].double()[:, None]
        y = torch.nn.functional.linear(x, w)
        parts.append(y + s["bias"].double() if case["bias"] else y)
    return torch.cat(parts)


def _exact_append(case, s):
    D = case["head_dim"]
    positions = torch.cat([torch.arange(m - n, m) for n, m in zip(s["q_lens"], s["kv_lens"])]).cuda()
    k = _exact_turn(s["k"].double(), positions, D, 1e6, case["layout"] == "half")

    def held(x):
        x = x.unflatten(-1, (-1, 32))
        peak = torch.maximum(x.amax(-1), -x.amin(-1))[..., None]
        e = torch.floor(torch.log2(peak))
        e = e + (peak >= _power(e + 1)).double() - (peak < _power(e)).double()  # the logarithm's own rounding
        scale = _power(e - 2 + (peak / _power(e - 2) > 7).double())
        u = x / scale
        # one bit behind the leading one, down to steps of a half
        step = 0.5 + 0.5 * (u.abs() >= 2) + 1.0 * (u.abs() >= 4)
        return ((torch.round(u / step) * step).clamp(-6, 6) * scale).flatten(-2)

    return held(k), held(s["v"].double())


def _exact_attention(case, s):
    H, K, D, P = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    G, row, out = H // K, 0, []

    def value(code):  # sign, two bits of exponent, one of mantissa
        e, f = code >> 1 & 3, (code & 1).double()
        a = torch.where(e == 0, f / 2, (1 + f / 2) * _power(e.int() - 1))
        return torch.where(code >= 8, -a, a)

    for b, (lo, hi, sinks) in enumerate(_windows(case)):
        keys = int(hi.max())
        page = s["data"].view(s["pages"], K, -1)[s["table"][b, :(keys + P - 1) // P].long()]
        sides = []
        for values in (0, 1):
            codes = page[..., values * P * D // 2:(values + 1) * P * D // 2]
            scales = page[..., P * D + values * P * D // 32:][..., :P * D // 32]
            if values:
                codes = codes.reshape(-1, K, P // 4, 16, 4, D // 32).permute(0, 1, 2, 4, 3, 5)
            codes = codes.reshape(-1, K, P, D // 2, 1)
            x = torch.cat([value(codes & 15), value(codes >> 4)], -1).reshape(-1, K, P, D // 32, 32)
            scales = scales.reshape(-1, K, P // 8, D // 32, 8).permute(0, 1, 2, 4, 3).reshape(-1, K, P, D // 32, 1)
            x = x * _power(scales.int() - 127)
            sides.append(x.reshape(-1, K, P, D).transpose(0, 1).reshape(K, -1, D)[:, :keys])
        for at in range(0, len(lo), 512):
            a, z, first = (t[at:at + 512, None].cuda() for t in (lo, hi, sinks))
            j = torch.arange(keys, device="cuda")
            hidden = (j >= z) | ((j < a) & (j >= first))
            q = s["q"][row + at:row + at + len(a)].double()
            o = torch.empty(len(a), H, D, dtype=torch.float64, device="cuda")
            for h in range(K):
                t = q[:, h * G:(h + 1) * G].transpose(0, 1) @ sides[0][h].t() / math.sqrt(D)
                o[:, h * G:(h + 1) * G] = (torch.softmax(t.masked_fill(hidden, -math.inf), -1) @ sides[1][h]).transpose(0, 1)
            out.append(o)
        row += len(lo)
    return torch.cat(out)
