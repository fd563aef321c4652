"""Where the attention block's operators can go wrong beside their ordinary
sizes: waves of one query inside tiles of several, caches of one row, peaks
that 32 bits do not tell apart, probabilities below half precision's normal
range."""
import math

import pytest
import torch

import operator_refs as ref
import test_gpu_operators as T
from nemo_amd import operators as ops

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("H,K,D,n,left,right", [
    (64, 32, 64, 305, 20, 0),     # 128 rows a tile: query 304 is alone in a wave
    (32, 8, 64, 649, 130, 0),     # the same with a group of 4
    (32, 1, 64, 600, 20, 5),      # 128 rows: a wave has one query, a tile four
    (40, 1, 128, 500, 20, 0),     # waves of one query and of two
    (64, 2, 64, 300, 20, 5),
    (32, 8, 128, 265, 400, 0),    # 64 rows in four parts: query 264 is alone
    (32, 1, 128, 300, 400, 3),    # the same: a wave has one query, a tile two
])
def test_attention_hidden_values_of_a_tile(torch_cuda, H, K, D, n, left, right, dtype):
    """Infinities and NaN in values that the last query does not see and the
    one before it does leave it, and all others that do not see them, as they
    are."""
    sinks, m = 2, n + 200
    b = T.Batch(dtype, H, K, D, left, right, sinks, [n], [m], poison=False)
    last = m - 1 - left - 1  # right before the last query's window
    bad = [last, last - 13]
    for j, value in zip(bad, (math.inf, math.nan)):
        b.v[j] = value
    b.dv = b.v.cuda()
    b.run()
    touched = ref.visible(n, m, left, right, sinks)[:, bad].any(1)
    assert touched[n - 2] and not touched[n - 1]
    out = b.out[:n]
    assert not torch.isfinite(out[touched].float()).any()
    want, tol = ref.attention(b.q, b.k[:m], torch.nan_to_num(b.v[:m], nan=0.0, posinf=0.0, neginf=0.0), left, right, sinks,
                              D ** -0.5)
    T.close(out[~touched], want[~touched], tol[~touched])


@pytest.mark.parametrize("dtype,D", [(F16, 64), (F16, 128), (BF16, 128)])
@pytest.mark.parametrize("row", [0, 64])
@pytest.mark.parametrize("H,K,q_lens", [(4, 2, [1]), (4, 2, [3, 1, 20]), (32, 8, [600, 1]), (32, 8, [260, 30])])
def test_attention_of_one_key_row(torch_cuda, H, K, q_lens, row, dtype, D):
    """A cache of a single row, which every request has, whatever the distance
    to a next row is said to be: the result is its value."""
    b = T.Batch(dtype, H, K, D, -1, -1, 0, q_lens, [1] * len(q_lens), poison=False)
    b.dk, b.dv = b.dk[:1], b.dv[:1]
    b.starts = [0] * len(q_lens)
    b.kv_start.zero_()
    args = b.args(max_kv=400)  # (a hint that reaches every kernel)
    assert args.kv_rows == 1
    args.k_row = args.v_row = row
    b.attention.run(args, T.stream())
    torch.cuda.synchronize()
    b.check()


def tied_row(dtype, type8, hidden, seed, with_delta):
    """x, delta and w of a row whose two largest products, in columns of two
    lanes of a wave, round to the same 32 bits and whose second is the larger
    one; the other columns' quotients lie between the borders of two codes that
    the two would give. Returns x, delta, w, products (64 bits)."""
    g = torch.Generator().manual_seed(seed)

    def products(targets):
        """h, delta and w whose products are the targets' nearest of some hundred."""
        t = targets.double()[:, None].expand(-1, 400)
        if with_delta:  # what 32 bits lose of the sum
            h = t.float()
            d, w = (t - h.double()).float(), torch.ones_like(h)
            return h, d, w, h.double() + d.double()
        h = (1 + torch.rand(t.shape, generator=g)).to(dtype)
        w = (t / h.double()).float()
        return h, torch.zeros_like(h), w, h.double() * w.double()

    top = 127.0 if type8 == ops.TYPE_I8 else 448.0
    P = 400.0 * (1 + 2.0 ** -10)
    h, d, w, p = products(torch.tensor([P, P * (1 + 2.0 ** -26)], dtype=torch.float64))
    if with_delta:
        first, second = (h[0, 0], d[0, 0], w[0, 0], p[0, 0]), (h[1, 0], d[1, 0], w[1, 0], p[1, 0])
    else:
        h, d, w, p = (t.flatten() for t in (h, d, w, p))
        same = (p.float() == torch.tensor(P).float()).nonzero().flatten()
        lo, hi = same[p[same].argmin()], same[p[same].argmax()]
        first, second = (tuple(t[i] for t in (h, d, w, p)) for i in (lo, hi))
    low, high = float(first[3]), float(second[3])
    assert low < high and torch.tensor(low).float() == torch.tensor(high).float()
    if type8 == ops.TYPE_I8:
        border = torch.arange(30, 126) + 0.5
    else:  # the middles between 8-bit floats
        border = torch.cat([(torch.arange(8, 16) + 0.5) * 2.0 ** e for e in range(-2, 5)])
    border = border.double()[torch.arange(hidden) % len(border)]
    a, b = low * border / top, high * border / top
    h, d, w, p = products((a + b) / 2)
    inside = (p > a[:, None]) & (p < b[:, None])
    pick = (p - ((a + b) / 2)[:, None]).abs().masked_fill(~inside, math.inf).argmin(1, keepdim=True)
    x, delta, weight, v, between = (t.gather(1, pick).flatten() for t in (h, d, w, p, inside))
    for column, (ph, pd, pw, pp) in ((1, first), (hidden // 4 // 8 * 8 % 512 + 9, second)):
        x[column], delta[column], weight[column], v[column], between[column] = ph, pd, pw, pp, False
    return x, delta, weight, v, between, high


@pytest.mark.parametrize("dtype,with_delta", [(F16, False), (F32, False), (F32, True)])
@pytest.mark.parametrize("type8", [ops.TYPE_I8, ops.TYPE_E4M3])
@pytest.mark.parametrize("hidden", [512, 1024, 4096, 8192, 16384, 32768, 1001])
def test_norm_codes_of_peaks_that_tie(torch_cuda, hidden, type8, dtype, with_delta):
    """A row's scale is that of its exactly largest product, where several
    round to the same 32 bits."""
    x, delta, w, v, between, peak = tied_row(dtype, type8, hidden, 81, with_delta)
    x, delta = x.to(dtype), delta.to(dtype)
    dx, dd, dw = x.cuda(), delta.cuda(), w.cuda()
    y8 = torch.empty(hidden, dtype=torch.int8 if type8 == ops.TYPE_I8 else torch.float8_e4m3fn, device="cuda")
    scale = torch.empty(1, device="cuda")
    ops.RmsNorm().run(ops.norm_args(T.CODE[dtype], 1, hidden, dx.data_ptr(), dw.data_ptr(), 1e-5,
                                    dd.data_ptr() if with_delta else 0, d_y8=y8.data_ptr(), type8=type8,
                                    d_scales=scale.data_ptr()), T.stream())
    torch.cuda.synchronize()
    u = v * (127.0 if type8 == ops.TYPE_I8 else 448.0) / peak
    unit = torch.ones_like(u) if type8 == ops.TYPE_I8 else torch.exp2(torch.floor(torch.log2(u.abs())) - 3)
    clear = ((u / unit) % 1 - 0.5).abs() > 2.0 ** -40
    assert (between & clear).sum() > hidden / 8
    assert torch.equal(y8.cpu().double()[clear], (torch.round(u / unit) * unit)[clear])


@pytest.mark.parametrize("hidden", [8, 9])
def test_norm_of_more_rows_than_a_launch_takes(torch_cuda, hidden):
    """Rows past 2^21 are another launch's; the sum replaces the residual, and
    outputs' rows have space between them."""
    rows = (1 << 21) + 7
    x, delta, w = T.rand(91, rows, hidden, dtype=F16), T.rand(92, rows, hidden, dtype=F16), 1 + 0.1 * T.rand(93, hidden)
    dx, dd, dw = x.cuda(), delta.cuda(), w.cuda()
    y = torch.full((rows, hidden + 8), 7.0, dtype=F16, device="cuda")
    y8 = torch.zeros(rows, hidden + 8, dtype=torch.int8, device="cuda")
    scales = torch.full((rows, 2), 7.0, device="cuda")
    ops.RmsNorm().run(ops.norm_args(ops.TYPE_F16, rows, hidden, dx.data_ptr(), dw.data_ptr(), 1e-5, dd.data_ptr(),
                                    dx.data_ptr(), y.data_ptr(), y8.data_ptr(), ops.TYPE_I8, scales.data_ptr(),
                                    y_row=hidden + 8, y8_row=hidden + 8, scales_row=2), T.stream())
    torch.cuda.synchronize()
    h, want, rel = ref.norm(x, delta, w, 1e-5)
    T.close(dx, h, (ref.HALF[F16] + 2.0 ** -24) * h.abs() + ref.TINY[F16], "sum")
    T.close(y[:, :hidden], want, (ref.HALF[F16] + rel) * want.abs() + ref.TINY[F16], "y")
    T.check8(y8[:, :hidden].contiguous(), scales[:, :1], want, rel, ops.TYPE_I8, 0)
    assert (y[:, hidden:] == 7.0).all() and not y8[:, hidden:].any() and (scales[:, 1] == 7.0).all()


@pytest.mark.parametrize("H,K,D,n,m", [(8, 1, 64, 1, 60000), (8, 1, 128, 1, 60000), (8, 2, 128, 40, 5000),
                                       (64, 32, 64, 300, 3000), (32, 8, 128, 300, 3000)])
def test_attention_in_half_precision_behind_a_strong_sink(torch_cuda, H, K, D, n, m):
    """The first key's score lies 17 above a long cache of even ones, each of
    which has e^-17 of its probability, and all of the result: the first
    value is 0.

    operator_refs.attention's bound with one term smaller: probabilities are
    taken against a reference at least 8 powers of two below the row's largest
    score, so their sum is 2^8 or more and those that are rounded by up to
    2^-25 whatever they are add 2^-33 (sum |v| + n |out|)."""
    b = T.Batch(F16, H, K, D, -1, 0, 1, [n], [m], poison=False)
    u = T.rand(51, D)
    b.q = (u + 0.01 * b.q.float()).half()
    b.k = (0.01 * b.k.float()).half()
    b.k[0] = (17 * D ** 0.5 / (u * u).sum() * u).half()
    b.v = (1 + 0.1 * b.v.float()).half()
    b.v[0] = 0
    b.dq, b.dk, b.dv = torch.cat([b.q, torch.zeros(3, H, D, dtype=F16)]).cuda(), b.k.cuda(), b.v.cuda()
    b.run()
    want, tol = ref.attention(b.q, b.k[:m], b.v[:m], -1, 0, 1, D ** -0.5)
    seen = ref.visible(n, m, -1, 0, 1).double()
    for h in range(H):
        small = ref.TINY[F16] * (seen @ b.v[:m, h * K // H].double().abs() + seen.sum(1, keepdim=True) * want[:, h].abs())
        tol[:, h] -= (1 - 2.0 ** -8) * small
    T.close(b.out[:n], want, tol)
