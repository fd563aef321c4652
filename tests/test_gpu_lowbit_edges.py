"""Edges of the low-bit operators: a cache's values next to what the type does
not hold, beside rows that a NaN reaches."""
import math

import pytest
import torch

import lowbit_refs as lref
import operator_refs as ref
from test_gpu_lowbit import BF16, F16, Pages, attend, close, rand

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
