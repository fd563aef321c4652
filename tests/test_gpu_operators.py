"""The attention block's operators (nemo_amd.operators) against their
definitions in 64 bits: rotary positions, the residual RMSNorm with 8-bit
output, attention with a sliding window and sinks."""
import math

import pytest
import torch

import operator_refs as ref
from nemo_amd import operators as ops

pytestmark = pytest.mark.gpu

CODE = {torch.float16: ops.TYPE_F16, torch.bfloat16: ops.TYPE_BF16, torch.float32: ops.TYPE_F32}
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def rand(seed, *shape, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype)


def stream():
    return torch.cuda.current_stream().cuda_stream


def close(got, want, tol, what=""):
    off = (got.double().cpu() - want).abs() - tol
    if not off.numel():
        return
    assert not torch.isnan(off).any(), f"{what}: NaN"
    assert off.max() <= 0, f"{what}: {int((off > 0).sum())} of {off.numel()} outside, by up to {float(off.max())}"


# ---- rotary positions ---------------------------------------------------------

SCALINGS = {
    "none": {},
    "linear": dict(scaling=ops.ROPE_LINEAR, factor=4.0),
    "yarn": dict(scaling=ops.ROPE_YARN, factor=16.0, original_positions=16384),
    "bands": dict(scaling=ops.ROPE_BANDS, factor=8.0, original_positions=8192),
}
REF_SCALING = {"none": {}, "linear": dict(factor=4.0), "yarn": dict(factor=16.0), "bands": dict(factor=8.0, original=8192)}


def make_rope(d, rotary, half, scaling, theta=1e6, **more):
    rope = ops.Rope(ops.rope_config(d, rotary_dim=rotary, theta=theta, layout=ops.ROPE_HALF if half else
                                    ops.ROPE_INTERLEAVED, **SCALINGS[scaling], **more))
    freq = ref.rope_frequencies(rotary or d, theta, scaling, **REF_SCALING[scaling])
    return rope, freq, 0.1 * math.log(16) + 1 if scaling == "yarn" else 1.0


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rows,heads,kv,d,rotary,scaling", [
    (1, 32, 8, 64, 0, "yarn"),        # one token
    (3, 4, 1, 128, 0, "bands"),
    (37, 6, 2, 96, 40, "linear"),     # part of the head; half of 20 values is no whole vector of 16-bit ones
    (700, 5, 5, 80, 32, "none"),      # many tokens, each thread several heads
    (515, 40, 0, 64, 64, "yarn"),     # no keys
    (9, 3, 1, 10, 6, "none"),         # no vector fits
    (5, 1, 1, 2, 2, "linear"),        # one pair
    (600, 3, 2, 1024, 1000, "bands"),
])
def test_rope(torch_cuda, dtype, half, rows, heads, kv, d, rotary, scaling):
    rope, freq, mag = make_rope(d, rotary, half, scaling)
    q, k = rand(1, rows, heads, d, dtype=dtype), rand(2, rows, kv, d, dtype=dtype)
    pos = torch.randint(-50, 1 << 22, (rows,), generator=torch.Generator().manual_seed(3))
    dq, dk, dpos = q.cuda(), k.cuda(), pos.cuda()
    oq, ok = torch.full_like(dq, math.nan), torch.full_like(dk, math.nan)
    rope.apply(CODE[dtype], ops.rope_heads(dq.data_ptr(), oq.data_ptr(), heads, d),
               ops.rope_heads(dk.data_ptr(), ok.data_ptr(), kv, d) if kv else None, rows, dpos.data_ptr(),
               stream=stream())
    torch.cuda.synchronize()
    close(oq, *ref.rope(q, pos, freq, half, mag), "q")
    if kv:
        close(ok, *ref.rope(k, pos, freq, half, mag), "k")


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("shift", [0, 1])
def test_rope_in_place_in_projection_rows(torch_cuda, half, shift):
    """Query and key heads turned where they stand in rows of a projection,
    positions counted from `base`; value heads and other rows stay. Shifted by
    one element the rows fit no vector."""
    d, H, K, rows = 64, 6, 2, 41
    width = (H + 2 * K) * d + 8
    rope, freq, mag = make_rope(d, 0, half, "yarn")
    flat = rand(5, rows * width + 8, dtype=F16)
    dev = flat.cuda()
    x = dev.data_ptr() + 2 * shift
    heads = ops.rope_heads(x, x, H + K, d, x_row=width)
    rope.apply(ops.TYPE_F16, heads, None, rows - 1, base=1000, stream=stream())
    torch.cuda.synchronize()
    got = dev.cpu()
    before = flat[shift:shift + rows * width].view(rows, width)
    after = got[shift:shift + rows * width].view(rows, width)
    turned = before[:-1, :(H + K) * d].reshape(rows - 1, H + K, d)
    close(after[:-1, :(H + K) * d].reshape(rows - 1, H + K, d),
          *ref.rope(turned, torch.arange(rows - 1) + 1000, freq, half, mag))
    assert torch.equal(after[:, (H + K) * d:], before[:, (H + K) * d:]) and torch.equal(after[-1], before[-1])


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rows", [3, 600])
@pytest.mark.parametrize("d,rotary,shift,pad", [(128, 102, 0, 0), (128, 40, 0, 0), (128, 72, 4, 8), (64, 64, 2, 2), (64, 36, 1, 1),
                                                (160, 80, 0, 4), (300, 300, 0, 0), (6, 2, 0, 0)])
def test_rope_by_narrower_vectors(torch_cuda, dtype, half, rows, d, rotary, shift, pad):
    """Sizes, addresses and strides that leave vectors of 8, 4, 2 and 1 values;
    space between the rows stays."""
    heads, width = 5, 5 * d + pad
    rope, freq, mag = make_rope(d, rotary, half, "linear")
    x = rand(8, rows * width + 16, dtype=dtype).cuda()
    y = torch.full_like(x, 7.0)
    size = x.element_size() * shift
    rope.apply(CODE[dtype], ops.rope_heads(x.data_ptr() + size, y.data_ptr() + size, heads, d, x_row=width), None, rows, base=77,
               stream=stream())
    torch.cuda.synchronize()
    turned, out = (t[shift:shift + rows * width].view(rows, width).cpu() for t in (x, y))
    close(out[:, :heads * d].reshape(rows, heads, d),
          *ref.rope(turned[:, :heads * d].reshape(rows, heads, d), torch.arange(rows) + 77, freq, half, mag))
    assert (out[:, heads * d:] == 7.0).all() and (y[:shift] == 7.0).all() and (y[shift + rows * width:] == 7.0).all()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rotary", [40, 102, 32])
def test_rope_part_of_a_head_in_place(torch_cuda, half, rotary):
    """The rest of a head stays bit for bit, NaN with it; queries in place
    beside keys that go elsewhere."""
    rope, freq, mag = make_rope(128, rotary, half, "none")
    q, k = rand(9, 300, 4, 128, dtype=F16), rand(10, 300, 2, 128, dtype=F16)
    q[:, :, rotary:] = math.nan
    for elsewhere in (False, True):
        dq, dk = q.cuda(), k.cuda()
        ok = torch.zeros_like(dk) if elsewhere else dk
        rope.apply(ops.TYPE_F16, ops.rope_heads(dq.data_ptr(), dq.data_ptr(), 4, 128),
                   ops.rope_heads(dk.data_ptr(), ok.data_ptr(), 2, 128), 300, stream=stream())
        torch.cuda.synchronize()
        want, tol = ref.rope(torch.nan_to_num(q), torch.arange(300), freq, half, mag)
        close(dq[..., :rotary], want[..., :rotary], tol[..., :rotary] if torch.is_tensor(tol) else tol)
        assert torch.isnan(dq[..., rotary:]).all()
        close(ok, *ref.rope(k, torch.arange(300), freq, half, mag))


def test_rope_turns_back(torch_cuda):
    """By a position and by its negative gives the values back, but for two
    roundings of pairs (a, b): each of a + b's magnitude."""
    rope, freq, _ = make_rope(128, 0, True, "none")
    x = rand(7, 60, 4, 128).cuda()
    pos = (torch.arange(60) * 1237).cuda()
    neg = -pos
    y = x.clone()
    for p in (pos, neg):
        heads = ops.rope_heads(y.data_ptr(), y.data_ptr(), 4, 128)
        rope.apply(ops.TYPE_F32, heads, None, 60, p.data_ptr(), stream=stream())
    torch.cuda.synchronize()
    both = x[..., :64].abs() + x[..., 64:].abs()
    assert ((y - x).abs() <= 40 * 2.0 ** -24 * torch.cat([both, both], -1)).all()


def test_rope_of_nothing_and_head_strides(torch_cuda):
    """No rows and no heads are no work; heads may lie apart and in reverse
    order of rows and heads (head-major)."""
    rope, freq, mag = make_rope(64, 0, False, "none")
    x = rand(8, 3, 20, 64, dtype=BF16)  # [heads, rows, d]
    dx = x.cuda()
    dy = torch.zeros_like(dx)
    rope.apply(ops.TYPE_BF16, ops.rope_heads(dx.data_ptr(), dy.data_ptr(), 3, 64), None, 0, stream=stream())
    rope.apply(ops.TYPE_BF16, ops.rope_heads(0, 0, 0, 64), None, 20, stream=stream())
    torch.cuda.synchronize()
    assert not dy.any()
    rope.apply(ops.TYPE_BF16, ops.rope_heads(dx.data_ptr(), dy.data_ptr(), 3, 64, x_row=64, x_head=20 * 64), None, 20,
               stream=stream())
    torch.cuda.synchronize()
    close(dy.transpose(0, 1), *ref.rope(x.transpose(0, 1), torch.arange(20), freq, False, mag))


# ---- residual RMSNorm with 8-bit output ----------------------------------------

def check8(y8, scales, y, rel, type8, group):
    """Scales within the norm's error of max |y| / 127 or 448 (and one
    division); values within half a step of y (of y / scale: three more
    roundings in 32 bits), bytes' step the scale, 8-bit floats' 2^-4 of the
    value or 2^-10 scales."""
    rows, hidden = y.shape
    blocks = y.reshape(rows, -1, group or hidden)
    top = 127.0 if type8 == ops.TYPE_I8 else 448.0
    want = blocks.abs().amax(-1) / top
    s = scales.double().cpu()
    close(s, want, (rel + 2.0 ** -23) * want + 2.0 ** -149, "scales")
    values = y8.cpu().float().double().view(blocks.shape) * s[..., None]
    step = s[..., None] / 2 if type8 == ops.TYPE_I8 else torch.maximum(2.0 ** -4 * blocks.abs(), 2.0 ** -10 * s[..., None])
    close(values, blocks, step * (1 + 2.0 ** -20) + (rel + 2.0 ** -21) * blocks.abs(), "values")
    assert (y8.cpu().float().abs().view(blocks.shape).amax(-1)[want > 1e-38] == top).all()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("type8", [ops.TYPE_I8, ops.TYPE_E4M3])
@pytest.mark.parametrize("rows,hidden,group,shift", [
    (1, 2048, 0, 0), (5, 512, 128, 0), (2, 1, 0, 0), (3, 1001, 0, 0), (7, 4096, 64, 0), (4, 8192, 0, 0),
    (3, 96, 32, 0), (2, 16384, 128, 0), (2, 33280, 0, 0), (2, 33280, 128, 0), (9, 640, 64, 1), (300, 384, 0, 0),
    (2, 32768, 32, 0), (1, 8, 0, 0)])
def test_norm(torch_cuda, dtype, type8, rows, hidden, group, shift):
    """Every output, from rows of one value to rows that no register file
    holds; shifted by one element the buffers fit no vector."""
    x, delta, w = rand(11, rows, hidden, dtype=dtype), rand(12, rows, hidden, dtype=dtype), 1 + 0.1 * rand(13, hidden)
    if group and rows > 1:  # one group of zeros and one tiny group
        x[0, :group] = 0
        delta[0, :group] = 0
        w[hidden - group:] *= 2.0 ** -60
    flat = torch.empty(3, rows * hidden + 8, dtype=dtype).cuda()
    flat[0, shift:shift + rows * hidden] = x.reshape(-1).cuda()
    flat[1, shift:shift + rows * hidden] = delta.reshape(-1).cuda()
    views = [f[shift:shift + rows * hidden].view(rows, hidden) for f in flat]
    dx, dd, dsum = views
    y = torch.full((rows, hidden), math.nan, dtype=dtype, device="cuda")
    y8 = torch.empty(rows, hidden, dtype=torch.int8 if type8 == ops.TYPE_I8 else torch.float8_e4m3fn, device="cuda")
    scales = torch.full((rows, hidden // group if group else 1), math.nan, device="cuda")
    dw = w.cuda()
    ops.RmsNorm().run(ops.norm_args(CODE[dtype], rows, hidden, dx.data_ptr(), dw.data_ptr(), 1e-5, dd.data_ptr(),
                                    dsum.data_ptr(), y.data_ptr(), y8.data_ptr(), type8, scales.data_ptr(), group),
                      stream())
    torch.cuda.synchronize()
    h, want, rel = ref.norm(x, delta, w, 1e-5)
    close(dsum, h, (ref.HALF[dtype] + 2.0 ** -24) * h.abs() + ref.TINY[dtype], "sum")
    close(y, want, (ref.HALF[dtype] + rel) * want.abs() + ref.TINY[dtype], "y")
    check8(y8, scales, want, rel, type8, group)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("type8", [ops.TYPE_I8, ops.TYPE_E4M3])
@pytest.mark.parametrize("rows,hidden,group", [(600, 512, 0), (300, 4096, 64), (150, 8192, 0), (40, 16384, 128), (300, 1000, 0),
                                               (20, 12296, 0), (20, 20008, 0), (90, 131, 0), (70, 1001, 0), (60, 3145, 0),
                                               (30, 7003, 0), (9, 16383, 0), (5, 16385, 0)])
def test_norm_codes_are_those_of_64_bits(torch_cuda, dtype, type8, rows, hidden, group):
    """A code is round(h w top / max |h w|) in 64 bits, the sum x + delta
    included: values are left out whose quotient is within 2^-40 of a border
    between two codes, and 16-bit ones whose sum 32 bits do not hold (of which
    the rest of a group depends on at most the largest)."""
    x, delta, w = rand(61, rows, hidden, dtype=dtype), rand(62, rows, hidden, dtype=dtype), 1 + 0.1 * rand(63, hidden)
    dx, dd, dw = x.cuda(), delta.cuda(), w.cuda()
    y8 = torch.empty(rows, hidden, dtype=torch.int8 if type8 == ops.TYPE_I8 else torch.float8_e4m3fn, device="cuda")
    scales = torch.empty(rows, hidden // group if group else 1, device="cuda")
    ops.RmsNorm().run(ops.norm_args(CODE[dtype], rows, hidden, dx.data_ptr(), dw.data_ptr(), 1e-5, dd.data_ptr(),
                                    d_y8=y8.data_ptr(), type8=type8, d_scales=scales.data_ptr(), group=group), stream())
    torch.cuda.synchronize()
    h = x.double() + delta.double()
    held = torch.ones_like(h, dtype=torch.bool) if dtype == F32 else h == h.float().double()
    v = (h * w.double()).view(rows, -1, group or hidden)
    held = held.view(v.shape)
    held &= held.gather(-1, v.abs().argmax(-1, keepdim=True))
    u = v * (127.0 if type8 == ops.TYPE_I8 else 448.0) / v.abs().amax(-1, keepdim=True)
    unit = torch.ones_like(u) if type8 == ops.TYPE_I8 else torch.exp2(
        torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 3)  # the codes' distance
    steps = u / unit
    clear = ((steps.abs() % 1 - 0.5).abs() > 2.0 ** -40) & held
    got = y8.cpu().float().double().view(u.shape)
    assert clear.double().mean() > 0.99
    assert torch.equal(got[clear], (torch.round(steps) * unit)[clear])


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("hidden,group", [(384, 32), (512, 128), (1920, 64), (3968, 128), (4160, 64), (16256, 128), (16512, 32)])
def test_norm_of_unaligned_rows_in_place(torch_cuda, dtype, hidden, group):
    """Rows that begin anywhere, with space between them; the sum replaces the residual."""
    rows = 6
    x, delta, w = rand(65, rows, hidden, dtype=dtype), rand(66, rows, hidden, dtype=dtype), 1 + 0.1 * rand(67, hidden)
    stride = hidden + 3
    dx = torch.zeros(rows * stride + 1, dtype=dtype).cuda()[1:].view(rows, stride)
    dd = torch.zeros_like(dx)
    dx[:, :hidden], dd[:, :hidden] = x.cuda(), delta.cuda()
    dw = torch.zeros(hidden + 1).cuda()[1:]
    dw.copy_(w)
    y8 = torch.zeros(rows, stride, dtype=torch.int8, device="cuda")
    scales = torch.zeros(rows, hidden // group, device="cuda")
    y = torch.full((rows, stride), 7.0, dtype=dtype, device="cuda")
    ops.RmsNorm().run(ops.norm_args(CODE[dtype], rows, hidden, dx.data_ptr(), dw.data_ptr(), 1e-5, dd.data_ptr(), dx.data_ptr(),
                                    y.data_ptr(), y8.data_ptr(), ops.TYPE_I8, scales.data_ptr(), group, x_row=stride,
                                    delta_row=stride, sum_row=stride, y_row=stride, y8_row=stride), stream())
    torch.cuda.synchronize()
    h, want, rel = ref.norm(x, delta, w, 1e-5)
    close(dx[:, :hidden], h, (ref.HALF[dtype] + 2.0 ** -24) * h.abs() + ref.TINY[dtype], "sum")
    close(y[:, :hidden], want, (ref.HALF[dtype] + rel) * want.abs() + ref.TINY[dtype], "y")
    check8(y8[:, :hidden], scales, want, rel, ops.TYPE_I8, group)
    assert not dx[:, hidden:].any() and (y[:, hidden:] == 7.0).all() and not y8[:, hidden:].any()


def test_norm_in_place_and_parts(torch_cuda):
    """The sum replaces the residual and y the branch; each output alone gives
    the same bits; padded rows keep their padding."""
    rows, hidden, pad = 6, 1536, 16
    x, delta, w = rand(21, rows, hidden + pad, dtype=F16), rand(22, rows, hidden, dtype=F16), rand(23, hidden)
    dx, dd, dw = x.cuda(), delta.cuda(), w.cuda()
    run = ops.RmsNorm().run
    y = torch.empty_like(dd)
    run(ops.norm_args(ops.TYPE_F16, rows, hidden, dx.data_ptr(), dw.data_ptr(), 1e-6, dd.data_ptr(), d_y=y.data_ptr(),
                      x_row=hidden + pad), stream())
    y8, s = torch.empty(rows, hidden, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    run(ops.norm_args(ops.TYPE_F16, rows, hidden, dx.data_ptr(), dw.data_ptr(), 1e-6, dd.data_ptr(),
                      d_y8=y8.data_ptr(), d_scales=s.data_ptr(), x_row=hidden + pad), stream())
    h, want, rel = ref.norm(x[:, :hidden], delta, w, 1e-6)
    torch.cuda.synchronize()
    check8(y8, s[:, None], want, rel, ops.TYPE_I8, 0)
    run(ops.norm_args(ops.TYPE_F16, rows, hidden, dx.data_ptr(), dw.data_ptr(), 1e-6, dd.data_ptr(),
                      d_sum=dx.data_ptr(), d_y=dd.data_ptr(), x_row=hidden + pad, sum_row=hidden + pad), stream())
    torch.cuda.synchronize()
    assert torch.equal(dd, y)
    close(dd, want, (ref.HALF[F16] + rel) * want.abs() + ref.TINY[F16], "y")
    close(dx[:, :hidden], h, (ref.HALF[F16] + 2.0 ** -24) * h.abs() + ref.TINY[F16], "sum")
    assert torch.equal(dx[:, hidden:].cpu(), x[:, hidden:])


@pytest.mark.parametrize("hidden", [256, 1000, 1001])
def test_norm_without_delta_and_weight_zero_and_nan_rows(torch_cuda, hidden):
    """A row of zeros gives zeros with scale 0; a NaN spoils its own row's
    scale and no other row."""
    x = rand(31, 4, hidden)
    x[1] = 0
    x[2, 5] = math.nan
    dx = x.cuda()
    y, y8, s = torch.empty_like(dx), torch.ones(4, hidden, dtype=torch.int8, device="cuda"), torch.empty(4, device="cuda")
    ops.RmsNorm().run(ops.norm_args(ops.TYPE_F32, 4, hidden, dx.data_ptr(), d_y=y.data_ptr(), d_y8=y8.data_ptr(),
                                    d_scales=s.data_ptr()), stream())
    torch.cuda.synchronize()
    assert s[1] == 0 and not y8[1].any() and not y[1].any()
    assert torch.isnan(s[2]) and torch.isnan(y[2]).all()
    keep = [0, 3]
    _, want, rel = ref.norm(x[keep], None, None, 1e-5)
    close(y[keep], want, (2.0 ** -24 + rel) * want.abs(), "y")
    check8(y8[keep], s[keep][:, None], want, rel, ops.TYPE_I8, 0)


# ---- attention with a sliding window and sinks ----------------------------------

class Batch:
    """Requests of a batch in a packed projection (kv_lens None) or a cache
    with room beyond every request, which NaN fills, as do all cache rows that
    no query sees. Queries and outputs have three rows behind the last request."""

    def __init__(self, dtype, H, K, D, left, right, sinks, q_lens, kv_lens=None, seed=41, poison=True):
        self.dtype, self.H, self.K, self.D, self.window = dtype, H, K, D, (left, right, sinks)
        self.q_lens, self.kv_lens = q_lens, q_lens if kv_lens is None else kv_lens
        rows = sum(q_lens)
        if kv_lens is None:
            self.qkv = rand(seed, rows, H + 2 * K, D, dtype=dtype)
            self.q, self.k, self.v = self.qkv[:, :H], self.qkv[:, H:H + K], self.qkv[:, H + K:]
            self.starts = [sum(q_lens[:i]) for i in range(len(q_lens))]
            dev = torch.cat([self.qkv, torch.zeros(3, H + 2 * K, D, dtype=dtype)]).cuda()
            self.dq, self.dk, self.dv = dev[:, :H], dev[:, H:H + K], dev[:, H + K:]
        else:
            cap = max(kv_lens) + 5
            self.q = rand(seed, rows, H, D, dtype=dtype)
            self.k, self.v = rand(seed + 1, len(q_lens) * cap, K, D, dtype=dtype), rand(seed + 2, len(q_lens) * cap, K, D, dtype=dtype)
            self.starts = [i * cap for i in range(len(q_lens))]
            if poison:
                seen = torch.zeros(len(self.k), dtype=torch.bool)
                for s, n, m in zip(self.starts, q_lens, kv_lens):
                    seen[s:s + m] = ref.visible(n, m, left, right, sinks).any(0)
                self.k[~seen] = math.nan
                self.v[~seen] = math.inf
            self.dq = torch.cat([self.q, torch.zeros(3, H, D, dtype=dtype)]).cuda()
            self.dk, self.dv = self.k.cuda(), self.v.cuda()
        self.out = torch.full((rows + 3, H, D), 7.0, dtype=dtype, device="cuda")
        starts = [sum(q_lens[:i]) for i in range(len(q_lens) + 1)]
        self.q_start = torch.tensor(starts, dtype=torch.int32).cuda()
        self.kv_start = torch.tensor(self.starts, dtype=torch.int64).cuda()
        self.kv_len = torch.tensor(self.kv_lens, dtype=torch.int32).cuda()

    def args(self, workspace=True, scale=0.0, max_kv=None):
        self.attention = ops.WindowAttention(ops.attention_config(
            self.H, self.K, self.D, CODE[self.dtype], *self.window, scale=scale))
        most = max(self.kv_lens) if max_kv is None else max_kv
        need = self.attention.workspace_bytes(len(self.q_lens), len(self.out), most) if workspace else 0
        self.workspace = torch.full((need + 1,), 0xff, dtype=torch.uint8, device="cuda")
        return ops.attention_batch(
            len(self.q_lens), len(self.out), len(self.dk), most, self.q_start.data_ptr(), self.kv_start.data_ptr(),
            self.kv_len.data_ptr(), *((t.data_ptr(), t.stride(0), t.stride(1)) for t in (self.dq, self.dk, self.dv, self.out)),
            d_workspace=self.workspace.data_ptr(), workspace_bytes=need)

    def run(self, **kw):
        args = self.args(**kw)
        self.attention.run(args, stream())
        torch.cuda.synchronize()
        return self

    def check(self, scale=None):
        row = 0
        for n, m, s in zip(self.q_lens, self.kv_lens, self.starts):
            want, tol = ref.attention(self.q[row:row + n], self.k[s:s + m], self.v[s:s + m], *self.window,
                                      scale or self.D ** -0.5)
            close(self.out[row:row + n], want, tol, f"request of {n} queries, {m} keys")
            row += n
        assert (self.out[row:] == 7.0).all(), "rows behind the last request"


WINDOWS = [(-1, -1, 0), (-1, 0, 0), (63, 0, 4), (0, 0, 0), (0, 0, 1), (130, 0, 70), (64, 64, 0), (31, 17, 200),
           (-1, 5, 0), (5, -1, 3), (1000, 1000, 1), (0, 0, 1000)]


# query and KV heads of batches that take the kernel for few rows and that for many
FEW_MANY = [(4, 2), (64, 32)]


@pytest.mark.parametrize("dtype,D", [(F16, 64), (F16, 128), (BF16, 64), (BF16, 128)])
@pytest.mark.parametrize("left,right,sinks", WINDOWS)
@pytest.mark.parametrize("H,K", FEW_MANY)
def test_attention_packed(torch_cuda, H, K, dtype, D, left, right, sinks):
    Batch(dtype, H, K, D, left, right, sinks, [1, 200, 0, 33, 257, 64]).run().check()


@pytest.mark.parametrize("dtype,D", [(F16, 64), (BF16, 128)])
def test_attention_many_requests(torch_cuda, dtype, D):
    """More requests than a wave has lanes, many of them empty or of one token."""
    lens = [(7 * i * i + 3 * i) % 23 for i in range(150)]
    Batch(dtype, 4, 1, D, 9, 0, 2, lens).run().check()
    Batch(dtype, 24, 8, D, 9, 2, 2, lens).run().check()
    Batch(dtype, 8, 8, D, 50, 0, 2, [min(1, n) for n in lens], [n * 11 for n in lens]).run().check()


@pytest.mark.parametrize("count", [64, 65, 128, 500, 4097, 4200])
def test_attention_numbers_of_requests(torch_cuda, count):
    """Around the numbers at which the search for a tile's request takes another round."""
    Batch(F16, 2, 1, 64, 9, 0, 1, [(5 * i * i + i) % 4 for i in range(count)]).run().check()


@pytest.mark.parametrize("dtype,D", [(F16, 64), (BF16, 128)])
@pytest.mark.parametrize("H,K", [(1, 1), (3, 1), (5, 1), (8, 1), (16, 2), (40, 1), (6, 6), (24, 8)])
def test_attention_head_groups(torch_cuda, dtype, D, H, K):
    Batch(dtype, H, K, D, 40, 0, 2, [70, 1, 19]).run().check()
    Batch(dtype, H, K, D, 300, 0, 2, [1, 2, 1], [700, 350, 1]).run().check()
    many = 520 * 32 // H  # rows for the kernel for many
    Batch(dtype, H, K, D, 40, 7, 2, [many - 300, 300 if many > 300 else 0] if many > 300 else [many]).run().check()


@pytest.mark.parametrize("dtype,D", [(F16, 64), (F16, 128), (BF16, 64), (BF16, 128)])
@pytest.mark.parametrize("left,right,sinks", [(-1, 0, 0), (1023, 0, 4), (63, 0, 0), (0, 0, 0), (100, 0, 130), (200, 3, 1)])
@pytest.mark.parametrize("workspace", [True, False])
def test_attention_one_token(torch_cuda, dtype, D, left, right, sinks, workspace):
    """Single tokens behind caches of all lengths; what they do not see holds
    NaN and infinities."""
    Batch(dtype, 8, 2, D, left, right, sinks, [1] * 7, [1, 64, 65, 5000, 2, 1024, 1090]).run(workspace=workspace).check()


@pytest.mark.parametrize("dtype,D", [(F16, 128), (BF16, 64)])
@pytest.mark.parametrize("left,right,sinks", [(-1, 0, 0), (255, 0, 4), (10, 0, 40)])
def test_attention_pieces(torch_cuda, dtype, D, left, right, sinks):
    """Several tokens behind a cache; requests without tokens, without keys,
    and with fewer keys than queries, whose first queries see nothing."""
    Batch(dtype, 4, 1, D, left, right, sinks, [5, 0, 100, 3, 40, 17], [900, 30, 700, 0, 25, 17]).run().check()
    Batch(dtype, 64, 16, D, left, right, sinks, [5, 0, 100, 3, 240, 17], [900, 30, 700, 0, 25, 17]).run().check()


@pytest.mark.parametrize("workspace", [True, False])
def test_attention_long_cache(torch_cuda, workspace):
    Batch(BF16, 8, 1, 128, -1, 0, 0, [1, 1], [70000, 3]).run(workspace=workspace).check()
    Batch(F16, 8, 4, 64, 16000, 0, 64, [3], [40000]).run(workspace=workspace).check()


def test_attention_scale_and_extreme_scores(torch_cuda):
    b = Batch(F16, 4, 2, 64, -1, 0, 0, [130])
    b.run(scale=0.5)
    b.check(scale=0.5)
    # scores of some thousands: the softmax is the largest key's value, and nothing overflows
    b = Batch(F16, 2, 1, 64, -1, -1, 0, [90], [90], poison=False)
    b.q *= 60
    b.k *= 60
    b.dq, b.dk = torch.cat([b.q, b.q[:3]]).cuda(), b.k.cuda()
    b.run(scale=1.0)
    b.check(scale=1.0)


@pytest.mark.parametrize("H,K", FEW_MANY)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_scores_that_rise_and_fall(torch_cuda, H, K, dtype):
    """Along the keys scores rise by thousands, fall and rise again, so that
    the reference of the probabilities has to follow; a huge score that a
    query does not see has no part in it."""
    n = 300
    b = Batch(dtype, H, K, 64, 150, 20, 3, [n], [n], poison=False)
    size = torch.cat([torch.linspace(0.01, 40, 100), torch.linspace(40, 0.01, 100), torch.linspace(0.01, 90, 100)])
    b.k = (b.k[:n] * size[:, None, None]).to(dtype)
    b.v = b.v[:n]
    b.dk, b.dv = b.k.cuda(), b.v.cuda()
    b.run().check()


@pytest.mark.parametrize("dtype,D", [(F16, 64), (BF16, 128)])
@pytest.mark.parametrize("H,K", FEW_MANY)
def test_attention_hidden_values_reach_no_result(torch_cuda, H, K, dtype, D):
    """Keys that some queries of a request see and others do not: NaN and
    infinities in them reach the results of the former alone."""
    left, right, sinks, n = 20, 0, 2, 300
    b = Batch(dtype, H, K, D, left, right, sinks, [n], [n], poison=False)
    bad = [7, 150, 299]
    for j, value in zip(bad, (math.nan, math.inf, -math.inf)):
        b.v[j] = value
        b.k[j, 0] = math.nan
    b.dk, b.dv = b.k.cuda(), b.v.cuda()
    b.run()
    touched = ref.visible(n, n, left, right, sinks)[:, bad].any(1)
    out = b.out[:n].cpu()
    assert not torch.isfinite(out[touched].float()).any()
    want, tol = ref.attention(b.q, *(torch.nan_to_num(t, nan=0.0, posinf=0.0, neginf=0.0) for t in (b.k[:n], b.v[:n])), left,
                              right, sinks, D ** -0.5)
    close(out[~touched], want[~touched], tol[~touched])


@pytest.mark.parametrize("H,K", FEW_MANY)
@pytest.mark.parametrize("key", [3, 200])
def test_attention_spoilt_queries_and_keys(torch_cuda, H, K, key):
    """A NaN in a query spoils that query, one in a key the queries that see
    it, and both leave the others as they are."""
    n = 280
    b = Batch(BF16, H, K, 64, 30, 5, 1, [n], [n], poison=False)
    b.run()
    clean = b.out.clone()
    b.q[100] = math.nan
    b.k[key] = math.nan
    b.dq, b.dk = torch.cat([b.q, b.q[:3]]).cuda(), b.k.cuda()
    b.out.fill_(7.0)
    b.run()
    bad = ref.visible(n, n, 30, 5, 1)[:, key].clone()
    bad[100] = True
    out = b.out[:n]
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], clean[:n][~bad])


# 32 query and 8 KV heads of 128, 260 to 500 queries of 384 keys and more: tiles whose keys are dealt to four parts
PARTS = dict(H=32, K=8, D=128)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("left,right,sinks", [(-1, -1, 0), (-1, 0, 0), (400, 0, 4), (383, 64, 0), (500, 17, 200), (-1, 5, 0),
                                              (5, -1, 3), (1000, 1000, 1), (0, 0, 1000)])
def test_attention_in_parts(torch_cuda, dtype, left, right, sinks):
    """Requests of fewer keys than parts have, without tokens, without keys."""
    Batch(dtype, *PARTS.values(), left, right, sinks, [1, 200, 0, 33, 57, 64]).run(max_kv=4000).check()
    Batch(dtype, *PARTS.values(), left, right, sinks, [5, 0, 100, 3, 240, 17], [900, 30, 700, 0, 25, 17]).run().check()
    Batch(dtype, *PARTS.values(), left, right, sinks, [300], [1333]).run().check()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_in_parts_scores_that_rise_and_fall(torch_cuda, dtype):
    b = Batch(dtype, *PARTS.values(), 450, 20, 3, [300], [700], poison=False)
    size = torch.cat([torch.linspace(0.01, 40, 250), torch.linspace(40, 0.01, 200), torch.linspace(0.01, 60, 250)])
    b.k = (b.k[:700] * size[:, None, None]).to(dtype)
    b.v = b.v[:700]
    b.dk, b.dv = b.k.cuda(), b.v.cuda()
    b.run().check()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_in_parts_spoilt_values(torch_cuda, dtype):
    """Infinite values, NaN queries and keys reach the queries that see them alone."""
    left, right, sinks, n, m = 500, 0, 2, 300, 900
    b = Batch(dtype, *PARTS.values(), left, right, sinks, [n], [m], poison=False)
    bad = [130, 899]
    for j, value in zip(bad, (math.inf, math.nan)):
        b.v[j] = value
    b.k[700] = math.nan
    b.q[30] = math.nan
    b.dq, b.dk, b.dv = torch.cat([b.q, b.q[:3]]).cuda(), b.k.cuda(), b.v.cuda()
    b.out.fill_(7.0)
    b.run()
    touched = ref.visible(n, m, left, right, sinks)[:, bad + [700]].any(1)
    touched[30] = True
    out = b.out[:n]
    assert not torch.isfinite(out[touched].float()).any()
    want, tol = ref.attention(torch.nan_to_num(b.q), *(torch.nan_to_num(t[:m], nan=0.0, posinf=0.0, neginf=0.0)
                                                       for t in (b.k, b.v)), left, right, sinks, 128 ** -0.5)
    close(out[~touched], want[~touched], tol[~touched])


def test_attention_cut_index_arrays(torch_cuda):
    """Entries outside the buffers are cut to them."""
    b = Batch(F16, 4, 2, 64, 50, 0, 0, [10, 6], [80, 60], poison=False)
    b.kv_len = torch.tensor([80, 1 << 30], dtype=torch.int32).cuda()  # the second runs to the buffer's end
    rows = len(b.dk)
    b.run()
    b.kv_lens = [80, rows - b.starts[1]]
    b.check()
    b.kv_start = torch.tensor([-5, 1 << 40], dtype=torch.int64).cuda()
    b.q_start = torch.tensor([0, 10, 1 << 30], dtype=torch.int32).cuda()
    b.kv_len = torch.tensor([-3, 9], dtype=torch.int32).cuda()
    b.run()
    assert not b.out.any()  # no keys: every row, the last three too, is 0


@pytest.mark.parametrize("H,K,D,keys", [(4, 2, 64, 300), (64, 32, 64, 300), (4, 2, 64, 3000), (32, 8, 128, 400)])
@pytest.mark.parametrize("q_start", [[0, 297, 5, 300], [290, 295, 0, 299], [300, 0, 300, 0], [0, -7, 200, 100]])
def test_attention_of_requests_out_of_order(torch_cuda, H, K, D, keys, q_start):
    """q_start that does not ascend says nothing about the results, but only
    rows of the buffers are read and written."""
    b = Batch(F16, H, K, D, -1, 0, 0, [5, 5, 5], [keys] * 3, poison=False)
    n = 300
    q, out = (torch.full((3 * n, H, D), 7.0, dtype=F16, device="cuda") for _ in range(2))
    b.dq, b.out = q[n:2 * n], out[n:2 * n]
    b.q_start = torch.tensor(q_start, dtype=torch.int32).cuda()
    b.run()
    assert (out[:n] == 7.0).all() and (out[2 * n:] == 7.0).all()


def test_attention_far_offsets(torch_cuda):
    """A cache whose last request starts past 2^32 bytes and 2^31 elements."""
    K, D = 8, 128
    rows = (1 << 31) // (K * D) + 700
    b = Batch(BF16, 8, K, D, 300, 0, 4, [1, 5], [600, 640], poison=False)
    big = torch.zeros(2, rows, K, D, dtype=BF16, device="cuda")
    at = [rows - 1300, rows - 641]
    for s, d, m in zip(b.starts, at, b.kv_lens):
        big[0, d:d + m], big[1, d:d + m] = b.dk[s:s + m], b.dv[s:s + m]
    b.dk, b.dv = big[0], big[1]
    b.kv_start = torch.tensor(at, dtype=torch.int64).cuda()
    b.run().check()


@pytest.mark.parametrize("H,K,n", [(4, 2, 60), (64, 32, 300)])
def test_attention_strides(torch_cuda, H, K, n):
    """Head-major caches, queries and outputs; keys that all heads share
    (stride 0 over heads)."""
    b = Batch(F16, H, K, 64, 100, 0, 3, [n, 9], [2 * n, 120], poison=False)
    b.k[:, 1:] = b.k[:, :1]
    b.dk = b.k[:, :1].cuda().expand(-1, K, -1)
    b.dv = b.v.cuda().transpose(0, 1).contiguous().transpose(0, 1)
    b.dq = b.dq.transpose(0, 1).contiguous().transpose(0, 1)
    b.out = torch.full((H, n + 12, 64), 7.0, dtype=F16, device="cuda").transpose(0, 1)
    b.run().check()


def test_attention_streams_and_graph(torch_cuda):
    """Captured once and replayed with other lengths and values, eager work of
    the same workspace between the replays; another stream."""
    b = Batch(BF16, 8, 2, 128, 500, 0, 4, [1] * 4, [3000, 10, 700, 3000], poison=False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    args = b.args()
    b.attention.run(args, side.cuda_stream)
    side.synchronize()
    b.check()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        b.attention.run(args, torch.cuda.current_stream().cuda_stream)
    for lens in ([2999, 11, 1, 2500], [1, 1, 1, 1], [3000, 3000, 0, 600]):
        b.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        b.kv_lens = lens
        b.out.fill_(7.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        b.check()
        replayed = b.out.clone()
        b.out.fill_(7.0)
        b.attention.run(args, stream())
        torch.cuda.synchronize()
        assert torch.equal(replayed, b.out)


def test_attention_on_two_streams_at_once(torch_cuda):
    """One object, two batches with a workspace each, in flight together; both
    captured into one graph on its one stream may share one."""
    a = Batch(F16, 8, 2, 64, 4000, 0, 4, [1] * 3, [6000, 3, 5000], seed=71, poison=False)
    b = Batch(F16, 8, 2, 64, 4000, 0, 4, [2] * 3, [5500, 40, 4000], seed=75, poison=False)
    one, two = a.args(), b.args()
    assert one.workspace_bytes and two.workspace_bytes
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        a.attention.run(one, streams[0].cuda_stream)
        a.attention.run(two, streams[1].cuda_stream)
    torch.cuda.synchronize()
    a.check()
    b.check()
    first = one if one.workspace_bytes >= two.workspace_bytes else two
    one.workspace = two.workspace = first.workspace
    one.workspace_bytes = two.workspace_bytes = first.workspace_bytes
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for args in (one, two):
            a.attention.run(args, torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        a.out.fill_(7.0)
        b.out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        a.check()
        b.check()


def test_attention_same_bits(torch_cuda):
    """The same call gives the same bits."""
    b = Batch(F16, 8, 2, 128, -1, 0, 0, [1, 130], [20000, 5000], poison=False).run()
    first = b.out.clone()
    for _ in range(3):
        b.out.fill_(7.0)
        b.run()
        assert torch.equal(first, b.out)


def test_a_layer_of_operators(torch_cuda):
    """norm -> projection -> rotary -> attention -> projection -> residual
    norm with 8-bit output, each on what the one before wrote, every stage
    against 64 bits on the same inputs."""
    import numpy as np

    import oracle
    import synth
    from nemo_amd import runtime as rt
    H, K, D, hidden = 8, 2, 64, 512
    width = (H + 2 * K) * D
    lens = [37, 1, 90]
    rows = sum(lens)
    x, w1, w2 = rand(61, rows, hidden, dtype=F16), 1 + 0.1 * rand(62, hidden), 1 + 0.1 * rand(63, hidden)
    raw = [synth.quantize_q4k(0.04 * synth.normal(seed, n).reshape(-1, 256))
           for seed, n in ((64, width * hidden), (65, hidden * H * D))]
    weights = [rt.QuantWeight(rt.TYPE_Q4_K, width, hidden, raw[0].tobytes()),
               rt.QuantWeight(rt.TYPE_Q4_K, hidden, H * D, raw[1].tobytes())]
    dense = [torch.from_numpy(np.asarray(oracle.dequantize(12, r), dtype=np.float64)) for r in raw]
    dx, dw1, dw2 = x.cuda(), w1.cuda(), w2.cuda()
    empty = lambda *s, dtype=F16: torch.empty(*s, dtype=dtype, device="cuda")
    n1, qkv, att, proj = empty(rows, hidden), empty(rows, width), empty(rows, H * D), empty(rows, hidden)
    y8, s8 = empty(rows, hidden, dtype=torch.int8), empty(rows, dtype=F32)
    norm = ops.RmsNorm()
    rope, freq, mag = make_rope(D, 32, True, "linear", theta=1e4)
    positions = torch.cat([torch.arange(n) for n in lens])
    dpos = positions.cuda()
    starts = [0, 37, 38, 128]
    q_start = torch.tensor(starts, dtype=torch.int32).cuda()
    kv_start, kv_len = torch.tensor(starts[:3]).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    attention = ops.WindowAttention(ops.attention_config(H, K, D, left=16, right=16, sinks=1))
    st = stream()
    norm.run(ops.norm_args(ops.TYPE_F16, rows, hidden, dx.data_ptr(), dw1.data_ptr(), d_y=n1.data_ptr()), st)
    weights[0].matmul(n1.data_ptr(), rows, qkv.data_ptr(), stream=st)
    projected = qkv.clone()
    heads = ops.rope_heads(qkv.data_ptr(), qkv.data_ptr(), H + K, D, x_row=width)
    rope.apply(ops.TYPE_F16, heads, None, rows, dpos.data_ptr(), stream=st)
    at = qkv.data_ptr()
    attention.run(ops.attention_batch(3, rows, rows, 90, q_start.data_ptr(), kv_start.data_ptr(), kv_len.data_ptr(),
                                      (at, width, D), (at + 2 * H * D, width, D), (at + 2 * (H + K) * D, width, D),
                                      (att.data_ptr(), H * D, D)), st)
    weights[1].matmul(att.data_ptr(), rows, proj.data_ptr(), stream=st)
    before = proj.clone()
    norm.run(ops.norm_args(ops.TYPE_F16, rows, hidden, dx.data_ptr(), dw2.data_ptr(), d_delta=proj.data_ptr(),
                           d_sum=dx.data_ptr(), d_y8=y8.data_ptr(), d_scales=s8.data_ptr()), st)
    torch.cuda.synchronize()
    _, want, rel = ref.norm(x, None, w1, 1e-5)
    close(n1, want, (ref.HALF[F16] + rel) * want.abs() + ref.TINY[F16], "norm")
    for got, inp, wt in ((projected, n1, dense[0].view(width, hidden)), (before, att, dense[1].view(hidden, H * D))):
        want = inp.cpu().double() @ wt.T
        assert (got.cpu().double() - want).norm() <= 1e-2 * want.norm()  # the products' own bound
    got = qkv.cpu().view(rows, -1, D)
    source = projected.cpu().view(rows, -1, D)
    close(got[:, :H + K], *ref.rope(source[:, :H + K], positions, freq, True), "rotary")
    assert torch.equal(got[:, H + K:], source[:, H + K:])
    for a, b in zip(starts, starts[1:]):
        part = got[a:b]
        close(att[a:b].view(b - a, H, D), *ref.attention(part[:, :H], part[:, H:H + K], part[:, H + K:], 16, 16, 1,
                                                         D ** -0.5), "attention")
    h, want, rel = ref.norm(x, before.cpu(), w2, 1e-5)
    close(dx, h, (ref.HALF[F16] + 2.0 ** -24) * h.abs() + ref.TINY[F16], "residual")
    check8(y8, s8[:, None], want, rel, ops.TYPE_I8, 0)
