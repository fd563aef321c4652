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
