"""Edges of the low-bit operators: a cache's values next to what the type does
not hold, beside rows that a NaN reaches; the largest pages; buffers, rows,
heads and tables of which what counts lies past 2^32 bytes; hints that are too
short; calls at once on two streams."""
import math

import pytest
import torch

import lowbit_refs as lref
import operator_refs as ref
import test_gpu_lowbit as lowbit
from nemo_amd import operators as ops
from test_gpu_lowbit import (BF16, CODE, F16, F32, Pages, attend, check, close, rand, random_cache, rows8, side, starts,
                             stream)

pytestmark = pytest.mark.gpu

# (dim, KV heads, heads of a group, queries, keys, keys before a query): tiles of 16, 32 and 128 rows; the second one's
# keys are dealt to workgroups
SHAPES = [
    (64, 2, 4, 8, 160, 100), (128, 2, 4, 8, 160, 100), (64, 2, 3, 2, 4500, -1), (128, 1, 4, 40, 170, 60),
    (64, 2, 2, 70, 200, 90), (64, 512, 1, 256, 300, 120), (128, 256, 1, 256, 300, 120),
]


def largest_code(dtype, byte):
    """The largest magnitude code that is finite in `dtype` under a scale byte."""
    values = torch.tensor(lref.LEVELS, dtype=torch.float64) * 2.0 ** (byte - 127)
    return int(torch.isfinite(values.to(dtype).double()).sum()) - 1


def cache_of_large_values(dtype, n, heads, dim, seed):
    """Codes and scales whose scores are small (sums of probabilities are near
    the number of keys), with blocks of V whose scale byte is one that some codes
    overflow under: all of theirs are finite. Those of bf16 hold one value that is not
    zero, so that no column's sum overflows 32 bits."""
    g = torch.Generator().manual_seed(seed)
    kc, vc = (torch.randint(0, 16, (n, heads, dim), generator=g).to(torch.uint8) for _ in range(2))
    ks = torch.randint(118, 122, (n, heads, dim // 32), generator=g).to(torch.uint8)
    vs = torch.randint(124, 129, (n, heads, dim // 32), generator=g).to(torch.uint8)
    bytes_ = [141, 142, 143, 144, 200, 254] if dtype == F16 else [253, 254, 253, 254, 253, 254]
    for h in {0, heads - 1}:
        for i, byte in enumerate(bytes_):
            t, block = (7 + i * (n // 6)) % n, i % (dim // 32)
            most, at = largest_code(dtype, byte), slice(32 * block, 32 * block + 32)
            codes = torch.randint(0, most + 1, (32,), generator=g)
            if dtype == BF16:
                codes = torch.where(torch.arange(32) == 3 + i, torch.tensor(most), torch.tensor(0))
            vc[t, h, at] = (codes + 8 * torch.randint(0, 2, (32,), generator=g)).to(torch.uint8)
            vs[t, h, block] = byte
    return kc, ks, vc, vs


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,kv,group,queries,keys,left", SHAPES)
@pytest.mark.parametrize("cause", ["query", "key", "value", "overflow"])
def test_large_values_beside_a_row_that_is_not_finite(torch_cuda, dtype, dim, kv, group, queries, keys, left, cause):
    """A NaN in a query, in a key or a value that some rows see, or a value that
    the type does not hold spoils what it reaches: of a query and a key whole
    rows, of a value's scale 32 columns, of a value that overflows its own. Large
    values that are finite stay so everywhere else."""
    kc, ks, vc, vs = cache_of_large_values(dtype, keys, kv, dim, keys + dim)
    k, v = lref.decode4(kc, ks), lref.decode4(vc, vs)
    q = (rand(3, queries, kv * group, dim) / 64).to(dtype)
    see = ref.visible(queries, keys, left, 0, 2)
    heads = [h * group + i for h in sorted({0, kv - 1}) for i in range(group)]
    bad = torch.zeros(queries, kv * group, dim, dtype=torch.bool)
    h = kv - 1
    of_head = slice(h * group, h * group + group)
    t = keys - max(1, queries // 2)  # seen by the later half of the queries
    if cause == "query":
        q[queries // 2, h * group, 5] = math.nan
        bad[queries // 2, h * group] = True
    elif cause == "key":
        ks[t, h, 0] = 255
        bad[see[:, t], of_head] = True
    elif cause == "value":
        vs[t, h, 1] = 255
        v[t, h, 32:64] = 0
        bad[see[:, t], of_head, 32:64] = True
    else:
        byte = 141 if dtype == F16 else 253
        vs[t, h, 1], vc[t, h, 32:64] = byte, 8
        vc[t, h, 37] = largest_code(dtype, byte) + 1
        v[t, h, 32:64] = 0
        bad[see[:, t], of_head, 37] = True
    pages = Pages(kv, dim, 32, [keys])
    pages.put(0, kc, ks, vc, vs)
    out, need = attend(pages, q, [queries], left, 0, 2)
    assert (need > 0) == (keys > 4000)
    out, few = out.cpu()[:, heads], bad[:, heads]
    assert few.any() and not few.all()
    assert not torch.isfinite(out[few].float()).any()
    clean = torch.nan_to_num(q[:, heads].double())
    want, tol = ref.attention(clean.to(dtype), k[:, sorted({0, kv - 1})], v[:, sorted({0, kv - 1})], left, 0, 2,
                              dim ** -0.5)
    # The sum is that of the rounded probabilities p (1 + e), |e| <= eps / 2, so the quotient is off by the sum of p e (v -
    # out): eps / 2 of the sum of p |v|, which the tolerance has, and of |out|, which matters where one value is most of
    # it: that value's e and the others', which the denominator holds.
    tol = tol + ref.HALF[dtype] * want.abs()
    close(torch.where(few, want.to(dtype), out), want, tol)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,kv,group,queries,keys,left", SHAPES)
def test_a_nan_in_a_query_changes_no_other_row(torch_cuda, dtype, dim, kv, group, queries, keys, left):
    """Not in one bit, also where probabilities are far below the largest."""
    pages, _ = random_cache(keys + 1, [keys], kv, dim, 32)
    q = 3 * rand(3, queries, kv * group, dim).to(dtype)
    clean, _ = attend(pages, q, [queries], left, 0, 2)
    q[queries // 2, 0, 5] = math.nan
    out, _ = attend(pages, q, [queries], left, 0, 2)
    assert torch.isnan(out[queries // 2, 0]).all()
    out[queries // 2, 0] = clean[queries // 2, 0]
    assert torch.isfinite(clean.float()).all() and torch.equal(out, clean)


@pytest.mark.parametrize("dim,kv,group,queries,keys,left", SHAPES)
def test_the_largest_values(torch_cuda, dim, kv, group, queries, keys, left):
    """Every value of bf16's last two powers of two, all of one sign in half of the
    columns: each result is finite, the sums in front of the division are far above
    what 32 bits hold. (A lane's 8 keys, a wave's, and those of waves and pieces.)"""
    g = torch.Generator().manual_seed(keys)
    kc = torch.randint(0, 16, (keys, kv, dim), generator=g).to(torch.uint8)
    ks = torch.randint(118, 122, (keys, kv, dim // 32), generator=g).to(torch.uint8)
    vs = torch.randint(253, 255, (keys, kv, dim // 32), generator=g).to(torch.uint8)
    most = torch.where(vs == 253, largest_code(BF16, 253), largest_code(BF16, 254)).repeat_interleave(32, -1)
    vc = (torch.rand(keys, kv, dim, generator=g) * (most + 1)).floor().long()
    vc = torch.where(torch.arange(dim) % 2 == 0, most, vc + 8 * torch.randint(0, 2, vc.shape, generator=g)).to(torch.uint8)
    pages = Pages(kv, dim, 32, [keys])
    pages.put(0, kc, ks, vc, vs)
    some = sorted({0, kv - 1})
    k, v = lref.decode4(kc[:, some], ks[:, some]), lref.decode4(vc[:, some], vs[:, some])
    q = (rand(3, queries, kv * group, dim) / 64).to(BF16)
    heads = [h * group + i for h in some for i in range(group)]
    out, need = attend(pages, q, [queries], left, 0, 2)
    assert (need > 0) == (keys > 4000)
    want, tol = ref.attention(q[:, heads], k, v, left, 0, 2, dim ** -0.5)
    close(out[:, heads], want, tol + ref.HALF[BF16] * want.abs())  # (the sum's rounding, as above)


# ---- norms of heads --------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d", [64, 1024])
@pytest.mark.parametrize("power", [-55, 0, 58])
def test_norms_of_small_and_large_heads(torch_cuda, dtype, d, power):
    """Largest values from 2^-55, without an epsilon, to below 2^59."""
    rows, heads = 5, 3
    x = (torch.rand(rows, heads, d, generator=torch.Generator().manual_seed(power + 60)) * 1.8 - 0.9)
    x[..., 7], x[0] = 1.0, 1.9375
    x = (x.double() * 2.0 ** power).to(dtype)
    w = 1 + rand(2, d) / 4
    dx, dw = x.cuda(), w.cuda()
    out = torch.empty_like(dx)
    rope = ops.Rope(ops.rope_config(d, theta=1e4))
    rope.norm_apply(CODE[dtype], ops.rope_heads(dx.data_ptr(), out.data_ptr(), heads, d), None,
                    ops.head_norm(dw.data_ptr(), epsilon=0.0), rows, stream=stream())
    torch.cuda.synchronize()
    y, tol = lref.head_norm(x, w, 0.0, torch.arange(rows), ref.rope_frequencies(d, 1e4), False, 1.0)
    close(out, y, tol + ref.HALF[dtype] * y.abs() + ref.TINY[dtype])


# ---- pages -----------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,dim", [(F16, 64), (BF16, 128), (F32, 128)])
@pytest.mark.parametrize("page", [512, 1024])
def test_append_and_read_of_large_pages(torch_cuda, dtype, dim, page):
    lowbit.test_append_writes_the_documented_bytes(torch_cuda, dtype, 3, dim, page, [30, 0, 7, 1],
                                                   [page + 3, 5, 2 * page, 2 * page + 1])


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("page", [256, 512, 1024])
@pytest.mark.parametrize("dim,kv,group,q_lens,kv_lens,left,sinks", [
    (64, 2, 4, [1, 3], [1500, 2100], -1, 0), (128, 2, 4, [1, 2, 1], [513, 1025, 3000], 1030, 600),
    (128, 1, 4, [40], [1700], 700, 3), (64, 512, 1, [256], [1100], 600, 260), (128, 256, 1, [256], [600], -1, 0)])
def test_attention_over_large_pages(torch_cuda, dtype, page, dim, kv, group, q_lens, kv_lens, left, sinks):
    pages, held = random_cache(sum(kv_lens), kv_lens, kv, dim, page)
    q = rand(7, sum(q_lens), kv * group, dim, dtype=dtype)
    out, _ = attend(pages, q, q_lens, left, 0, sinks)
    check(out, held, q, q_lens, left, 0, sinks, kv_heads=sorted({0, kv - 1}))


# ---- past 2^32 bytes -------------------------------------------------------------------

FAR = 1 << 32
ROW = 1 << 23  # the largest stride


@pytest.fixture
def gigabytes(torch_cuda):
    """For tests of buffers that large: they are given back afterwards."""
    yield torch_cuda
    torch_cuda.cuda.empty_cache()


def far_pages(kv, dim, page, n):
    """A cache of one request whose pages all lie past 2^32 bytes."""
    pages = Pages(kv, dim, page, [n])
    per, first = (n + page - 1) // page, FAR // pages.cache.page_bytes + 1
    pages.count = first + per
    pages.data = torch.empty(pages.count, pages.cache.page_bytes, dtype=torch.uint8, device="cuda")
    pages.table[0, :per] = first + torch.randperm(per, generator=torch.Generator().manual_seed(n))
    pages.upload()
    return pages


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dim,kv,group,n,keys,page", [
    (128, 8, 4, 1, 2500, 1024), (64, 4, 3, 30, 300, 64), (128, 2, 4, 50, 200, 32), (64, 512, 1, 256, 300, 1024)])
def test_pages_past_4_gib(gigabytes, dtype, dim, kv, group, n, keys, page):
    """Appended, read and attended to, in tiles of 16, 32 and 128 rows."""
    pages = far_pages(kv, dim, page, keys)
    x = rand(5, 2, keys, kv, dim, dtype=dtype)
    dx, start = x.cuda(), starts([keys])
    pages.cache.append(pages.pages, ops.cache4_rows(CODE[dtype], keys, start.data_ptr(), side(dx[0]), side(dx[1])),
                       stream=stream())
    out = torch.empty(2, keys, kv, dim, device="cuda")
    pages.cache.read(pages.pages, ops.cache4_rows(ops.TYPE_F32, keys, start.data_ptr(), side(out[0]), side(out[1])),
                     stream=stream())
    some = sorted({0, kv - 1})
    torch.cuda.synchronize()
    codes, scales, _ = lref.encode4(x[:, :, some].double())
    held = lref.decode4(codes, scales)
    assert torch.equal(out[:, :, some].cpu().double(), held)
    q = rand(7, n, kv * group, dim, dtype=dtype)
    got, _ = attend(pages, q, [n])
    heads = [h * group + i for h in some for i in range(group)]
    want, tol = ref.attention(q[:, heads], held[0], held[1], -1, 0, 0, dim ** -0.5)
    close(got[:, heads], want, tol)


def far_rows(rows, heads, dim, dtype, row, head, offset=0):
    """Rows of heads in a buffer of their own, of which the last begins past 2^32 bytes."""
    n = (rows - 1) * row + (heads - 1) * head + dim
    assert n * torch.empty(0, dtype=dtype).element_size() > FAR
    flat = torch.empty(offset + n, dtype=dtype, device="cuda")
    return torch.as_strided(flat, (rows, heads, dim), (row, head, 1), offset)


# rows and heads that are the largest stride apart
FAR_ROWS = [(F16, 300, 2, ROW, 128), (F32, 150, 3, ROW, 128), (BF16, 3, 300, 128, ROW)]


@pytest.mark.parametrize("dtype,rows,heads,row,head", FAR_ROWS)
def test_rows_of_a_cache_past_4_gib(gigabytes, dtype, rows, heads, row, head):
    dim = 64
    x = rand(6, 2, rows, heads, dim, dtype=dtype)
    far = [far_rows(rows, heads, dim, dtype, row, head) for _ in range(2)]
    pages, start = Pages(heads, dim, 32, [rows]), starts([rows])
    for t, v in zip(far, x):
        t.copy_(v)
    rope = ops.Rope(ops.rope_config(dim, theta=1e4, layout=ops.ROPE_HALF))
    args = ops.cache4_rows(CODE[dtype], rows, start.data_ptr(), side(far[0]), side(far[1]))
    pages.cache.append(pages.pages, args, rope, stream=stream())
    torch.cuda.synchronize()
    for t in far:
        t.fill_(7.0)
    pages.cache.read(pages.pages, args, stream=stream())
    torch.cuda.synchronize()
    turned = lref.turn(x[0].double(), torch.arange(rows), ref.rope_frequencies(dim, 1e4), True)
    for got, v in zip(far, (turned, x[1].double())):
        codes, scales, margin = lref.encode4(v)
        differ = got.cpu().double() != lref.decode4(codes, scales)
        assert not (differ & (margin > 2.0 ** -32)).any()


@pytest.mark.parametrize("dtype,rows,heads,row,head", FAR_ROWS)
def test_norms_of_heads_past_4_gib(gigabytes, dtype, rows, heads, row, head):
    """Query heads in place, key heads to a buffer near by."""
    dim = 64
    x = far_rows(rows, heads, dim, dtype, row, head)
    host, w = rand(8, rows, heads, dim, dtype=dtype), 1 + rand(9, dim) / 4
    x.copy_(host)
    near, dw = torch.empty(rows, heads, dim, dtype=dtype, device="cuda"), w.cuda()
    rope = ops.Rope(ops.rope_config(dim, theta=1e4))
    for first in (True, False):
        keys = ops.rope_heads(x.data_ptr(), near.data_ptr(), heads, dim, row, head, heads * dim, dim)
        own = ops.rope_heads(x.data_ptr(), x.data_ptr(), heads, dim, row, head)
        rope.norm_apply(CODE[dtype], keys if first else own, None, ops.head_norm(dw.data_ptr()), rows, stream=stream())
    torch.cuda.synchronize()
    y, tol = lref.head_norm(host, w, 1e-5, torch.arange(rows), ref.rope_frequencies(dim, 1e4), False, 1.0)
    for got in (near, x):
        close(got, y, tol + ref.HALF[dtype] * y.abs() + ref.TINY[dtype])


@pytest.mark.parametrize("m,n,far", [(600, 40, "xy"), (40, 600, "w"), (1, 600, "w"), (600, 700, "xyw"),
                                     (2100, 8190, "xy"), (8190, 2100, "w")])
def test_products_of_rows_past_4_gib(gigabytes, m, n, far):
    k, dtype = 300, F16
    x, xs = rows8(1, m, k)
    w, ws = rows8(2, n, k)

    def placed(t, is_far):
        if not is_far:
            return t.cuda()
        at = torch.as_strided(torch.empty((t.shape[0] - 1) * ROW + t.shape[1], dtype=torch.int8, device="cuda"), t.shape,
                              (ROW, 1))
        return at.copy_(t)

    dx, dw, dxs, dws = placed(x, "x" in far), placed(w, "w" in far), xs.cuda(), ws.cuda()
    y_row = ROW if "y" in far else n
    y = torch.as_strided(torch.empty((m - 1) * y_row + n, dtype=dtype, device="cuda"), (m, n), (y_row, 1))
    ops.Matmul8().run(ops.matmul8_args(CODE[dtype], m, n, k, dx.data_ptr(), dxs.data_ptr(), dw.data_ptr(), dws.data_ptr(),
                                       y.data_ptr(), x_row=dx.stride(0), w_row=dw.stride(0), y_row=y_row), stream=stream())
    torch.cuda.synchronize()
    close(y, *lref.matmul8(x[:, :k], xs, w[:, :k], ws, None, dtype))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("kv,group,q_lens,row,head", [
    (2, 4, [1] * 300, ROW, 64), (1, 4, [300], ROW, 64), (512, 1, [300], ROW, 64), (300, 1, [2], 64, ROW),
    (1, 300, [3], 64, ROW)])
def test_queries_past_4_gib(gigabytes, dtype, kv, group, q_lens, row, head):
    """Rows and heads of q and out, in tiles of 16, 32 and 128 rows."""
    dim, rows, heads = 64, sum(q_lens), kv * group
    kv_lens = [20 + b % 50 if len(q_lens) > 1 else 320 for b in range(len(q_lens))]
    pages, held = random_cache(11, kv_lens, kv, dim, 32)
    q = rand(12, rows, heads, dim, dtype=dtype)
    dq, out = (far_rows(rows, heads, dim, dtype, row, head) for _ in range(2))
    dq.copy_(q)
    start = starts(q_lens)
    config = ops.attention_config(heads, kv, dim, CODE[dtype], right=0)
    pages.cache.attention(config, pages.pages, ops.cache4_queries(rows, max(kv_lens), start.data_ptr(), side(dq), side(out)),
                          stream=stream())
    torch.cuda.synchronize()
    check(out, held, q, q_lens, kv_heads=sorted({0, kv - 1}))


@pytest.mark.parametrize("queries", [1, 12])
def test_a_table_past_4_gib(gigabytes, queries):
    """Requests whose rows of the table are the largest apart."""
    count, dim, kv = 300, 64, 1
    kv_lens = [queries + b % 70 for b in range(count)]
    pages, held = random_cache(13, kv_lens, kv, dim, 32)
    table = torch.empty(count * ROW, dtype=torch.int32, device="cuda").view(count, ROW)
    table[:, :pages.table.shape[1]] = pages.d_table
    pages.pages.table, pages.pages.table_row = table.data_ptr(), ROW
    q_lens = [queries] * count
    rows = sum(q_lens)
    x = rand(14, 2, rows, kv, dim, dtype=F16)
    dx, start = x.cuda(), starts(q_lens)
    back = torch.empty(2, rows, kv, dim, device="cuda")
    pages.cache.append(pages.pages, ops.cache4_rows(ops.TYPE_F16, rows, start.data_ptr(), side(dx[0]), side(dx[1])),
                       stream=stream())
    pages.cache.read(pages.pages, ops.cache4_rows(ops.TYPE_F32, rows, start.data_ptr(), side(back[0]), side(back[1])),
                     stream=stream())
    q = rand(15, rows, 2, dim, dtype=F16)
    out, _ = attend(pages, q, q_lens)
    codes, scales, _ = lref.encode4(x.double())
    new = lref.decode4(codes, scales)
    assert torch.equal(back.cpu().double(), new)
    held = [tuple(torch.cat([t[:n - queries], new[i, b * queries:(b + 1) * queries]]) for i, t in enumerate(held[b]))
            for b, n in enumerate(kv_lens)]
    check(out, held, q, q_lens)


# ---- many requests ---------------------------------------------------------------------

def test_more_requests_than_two_searches_find(torch_cuda):
    """5000 requests, empty ones among them and rows that are nobody's at both ends: a wave
    looks at 64 at a time, here three times."""
    g = torch.Generator().manual_seed(3)
    count, dim, before = 5000, 64, 3
    kv_lens = torch.randint(0, 40, (count,), generator=g).tolist()
    q_lens = [min(n, m) for n, m in zip(torch.randint(0, 3, (count,), generator=g).tolist(), kv_lens)]
    pages = Pages(1, dim, 32, kv_lens)
    tokens, queries = sum(kv_lens), sum(q_lens)
    starts_of = [torch.cat([torch.zeros(1, dtype=torch.int64), torch.tensor(n).cumsum(0)]) + before for n in (kv_lens, q_lens)]
    starts_on = [t.int().cuda() for t in starts_of]
    x = rand(4, 2, tokens + 2 * before, 1, dim, dtype=F16)
    dx, back = x.cuda(), torch.full((2, tokens + 2 * before, 1, dim), 7.0, device="cuda")
    for call, kind, t in ((pages.cache.append, ops.TYPE_F16, dx), (pages.cache.read, ops.TYPE_F32, back)):
        call(pages.pages, ops.cache4_rows(kind, tokens + 2 * before, starts_on[0].data_ptr(), side(t[0]), side(t[1])),
             stream=stream())
    q = rand(5, queries + 2 * before, 2, dim, dtype=F16)
    out = torch.full(q.shape, 7.0, dtype=F16, device="cuda")
    attend(pages, q, None, out=out, start=starts_on[1])
    out, back = out.cpu(), back.cpu()
    for t in (out.unsqueeze(0), back):
        assert (t[:, :before] == 7.0).all() and (t[:, -before:] == 7.0).all()
    for b in [0, 1, 2, count - 2, count - 1] + torch.randperm(count, generator=g)[:200].tolist():
        (k0, k1), (q0, q1) = (t[b:b + 2].tolist() for t in starts_of)
        codes, scales, _ = lref.encode4(x[:, k0:k1].double())
        held = lref.decode4(codes, scales)
        assert torch.equal(back[:, k0:k1].double(), held)
        check(out[q0:q1], [(held[0], held[1])], q[q0:q1], [q1 - q0])


# ---- hints and streams -----------------------------------------------------------------

@pytest.mark.parametrize("dim,kv,group,q_lens,kv_lens,max_kv", [
    (64, 2, 3, [1, 2], [9000, 300], 2000), (128, 1, 4, [40], [5000], 2000), (64, 128, 1, [256], [5000], 4100)])
def test_a_hint_that_is_too_short(torch_cuda, dim, kv, group, q_lens, kv_lens, max_kv):
    """Pieces of a tile's keys grow where it has more than the hint says."""
    pages, held = random_cache(17, kv_lens, kv, dim, 64)
    q = rand(18, sum(q_lens), kv * group, dim, dtype=F16)
    out, need = attend(pages, q, q_lens, max_kv=max_kv)
    assert need > 0
    check(out, held, q, q_lens, kv_heads=sorted({0, kv - 1}))


def test_products_and_split_attention_on_two_streams(torch_cuda):
    """On streams of their own at once, with a workspace each: a product, an append
    of what it gives, and attention in pieces, again and again, equal the
    definitions."""
    H, K, D, hidden, rounds = 8, 2, 64, 512, 20
    w, ws = rows8(21, (H + 2 * K) * D, hidden)
    dw, dws, start = w.cuda(), ws.cuda(), starts([1])
    config, matmul8, sides = ops.attention_config(H, K, D, ops.TYPE_F16, right=0), ops.Matmul8(), []
    for i, n in enumerate((6000, 9000)):
        pages, held = random_cache(22 + i, [n], K, D, 64)
        need = pages.cache.workspace_bytes(config, 1, 1, n)
        assert need > 0
        x, xs = rows8(24 + i, 1, hidden)
        sides.append(dict(n=n, pages=pages, held=held, x=x, xs=xs, dx=x.cuda(), dxs=xs.cuda(), need=need,
                          space=torch.full((need,), 0xff, dtype=torch.uint8, device="cuda"),
                          qkv=torch.zeros(1, H + 2 * K, D, dtype=F16, device="cuda"),
                          out=torch.zeros(1, H, D, dtype=F16, device="cuda"), stream=torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(rounds):
        for s in sides:
            at, qkv = s["stream"].cuda_stream, s["qkv"]
            matmul8.run(ops.matmul8_args(ops.TYPE_F16, 1, (H + 2 * K) * D, hidden, s["dx"].data_ptr(), s["dxs"].data_ptr(),
                                         dw.data_ptr(), dws.data_ptr(), qkv.data_ptr()), stream=at)
            s["pages"].cache.append(s["pages"].pages, ops.cache4_rows(
                ops.TYPE_F16, 1, start.data_ptr(), side(qkv[:, H:H + K]), side(qkv[:, H + K:])), stream=at)
            s["pages"].cache.attention(config, s["pages"].pages, ops.cache4_queries(
                1, s["n"], start.data_ptr(), side(qkv[:, :H]), side(s["out"]), s["space"].data_ptr(), s["need"]), stream=at)
    torch.cuda.synchronize()
    for s in sides:
        qkv = s["qkv"].cpu()
        close(qkv.flatten(1), *lref.matmul8(s["x"], s["xs"], w, ws, None, F16))
        held = []
        for t, new in zip(s["held"][0], (qkv[:, H:H + K], qkv[:, H + K:])):
            codes, scales, _ = lref.encode4(new.double())
            held.append(torch.cat([t[:-1], lref.decode4(codes, scales)]))
        check(s["out"], [tuple(held)], qkv[:, :H], [1])
