"""What the library does around the operators' kernels, on a host whose HIP
runtime is tests/hip_on_host.c: failed passes and launch sizes, which no
device has to take part in. Each case runs in a process of its own, in which
the stand-in is loaded before the library."""
import os
import shutil
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))

PRELUDE = f"""
import ctypes, os, sys
sys.path[:0] = [{os.path.join(os.path.dirname(HERE), "nemotron-3-embed-webgpu_amd")!r}]
host = ctypes.CDLL(sys.argv[1], os.RTLD_GLOBAL | os.RTLD_NOW)
launches = ctypes.c_uint64.in_dll(host, "host_launches")
most_threads = ctypes.c_uint64.in_dll(host, "host_most_threads")
import numpy as np
from nemo_amd import _lib, operators as ops, runtime as rt
L = _lib.load()
"""


@pytest.fixture(scope="session")
def on_host(tmp_path_factory):
    """Runs a program against the stand-in; its output has to end in 'ok'."""
    cc = shutil.which("cc") or shutil.which("gcc")
    if cc is None:
        pytest.skip("needs a C compiler")
    lib = str(tmp_path_factory.mktemp("host") / "hip_on_host.so")
    subprocess.run([cc, "-O1", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-o", lib,
                    os.path.join(HERE, "hip_on_host.c")], check=True)

    def run(program):
        r = subprocess.run([sys.executable, "-c", PRELUDE + program, lib], capture_output=True, text=True, timeout=120)
        assert r.returncode == 0 and r.stdout.split()[-1:] == ["ok"], r.stdout[-2000:] + r.stderr[-2000:]

    return run


def test_token_states_of_a_failed_pass_are_refused(on_host):
    """A pass that fails before the merge leaves more rows than the merged
    stream has; wherever it fails, there are no token states until a pass has
    been enqueued to its end."""
    on_host("""
dims = rt.make_dims(hidden=256, q_heads=4, kv_heads=2, head_dim=64, intermediate=256, layers=4, vocab=300,
                    merge_after_layer=2)
model = rt.NemotronHipModel(None, dims=dims, synthetic_seed=3)
S, lens = 100, [100, 70]
plan = model.createPlan(2, S)
ids, n = np.ones(2 * S, np.uint32), sum(rt.contextual_merged_length(x) for x in lens)
y8, scales = np.empty(1000 * 256, np.int8), np.empty(1000, np.float32)

def states():
    return plan.token_states8(y8.ctypes.data, scales.ctypes.data, 1000)

def refused():
    before = launches.value
    try:
        got = states()
    except rt.NemoError as e:
        assert "has not run" in str(e), e
    else:
        raise AssertionError(f"{got} rows of token states")
    assert launches.value == before

refused()
out = np.empty((2, 256), np.float32)
failed = 0
while True:
    plan.run_sync(ids, lens)
    assert states() == n
    L.nemo_debug_fail_after(2 + failed)  # (the first check is hipSetDevice's)
    try:
        plan.run_device(ids.ctypes.data, lens, out.ctypes.data)
    except rt.NemoError as e:
        assert "injected" in str(e), e
        failed += 1
        refused()
    else:
        break
    finally:
        L.nemo_debug_fail_after(0)
assert states() == n and failed > 20, failed
plan.run_sync(ids, [3, 1])
assert states() == rt.contextual_merged_length(3) + rt.contextual_merged_length(1)
print("ok")
""")


@pytest.mark.parametrize("type_,hidden", [("TYPE_BF16", 2048), ("TYPE_BF16", 8192), ("TYPE_F32", 8192),
                                          ("TYPE_F16", 16384), ("TYPE_F32", 32768), ("TYPE_F16", 40001),
                                          ("TYPE_F16", 96)])
@pytest.mark.parametrize("rows", [1, (1 << 21) + 5, (1 << 23) - 1, 1 << 23])
def test_norm_grids_hold_their_rows(on_host, type_, hidden, rows):
    """The most rows that the norm takes, in grids below 2^32 threads, each
    row once: the launches' parts begin where the ones before end."""
    on_host(f"""
rows, hidden, type_ = {rows}, {hidden}, ops.{type_}
size = 4 if type_ == ops.TYPE_F32 else 2
at = {{"x": 1 << 40, "delta": 2 << 40, "sum": 3 << 40, "y": 4 << 40, "y8": 5 << 40, "scales": 6 << 40}}
args = ops.norm_args(type_, rows, hidden, at["x"], 7 << 40, 1e-5, at["delta"], at["sum"], at["y"], at["y8"],
                     ops.TYPE_I8, at["scales"])
parts = []
CALL = ctypes.CFUNCTYPE(None, ctypes.c_uint32, ctypes.c_uint32, ctypes.POINTER(_lib.NormArgs))

@CALL
def launched(grid, block, first):
    a = first.contents
    assert grid * block < 1 << 32 and 64 * a.rows <= grid * block, (grid, block, a.rows)
    parts.append((a.rows, a.x, a.delta, a.sum, a.y, a.y8, a.scales, a.weight))

ctypes.c_void_p.in_dll(host, "host_on_launch").value = ctypes.cast(launched, ctypes.c_void_p).value
ops.RmsNorm().run(args)
done = 0
for n, x, delta, sum_, y, y8, scales, weight in parts:
    assert [x, delta, sum_, y] == [at[k] + done * hidden * size for k in ("x", "delta", "sum", "y")]
    assert (y8, scales, weight) == (at["y8"] + done * hidden, at["scales"] + 4 * done, 7 << 40)
    done += n
assert done == rows and most_threads.value < 1 << 32, (done, most_threads.value)
print("ok")
""")


def test_attention_and_rope_grids(on_host):
    """The largest calls that are taken, by every kernel: grids below 2^32 threads."""
    on_host("""
A = 1 << 40
for heads, kv, dim in ((1, 1, 64), (32, 8, 128), (1024, 1, 64), (1024, 1024, 128), (4, 4, 128)):
    for count in (1, (1 << 22) // kv if kv >= 4 else 1 << 20):
        for max_kv in (1, 1000, 1 << 30):
            rows = (1 << 26) // heads
            a = ops.WindowAttention(ops.attention_config(heads, kv, dim))
            side = (A, heads * dim, dim)
            need = a.workspace_bytes(count, rows, max_kv)
            a.run(ops.attention_batch(count, rows, 1 << 30, max_kv, A, A, A, side, side, side, side, A, need))
            assert most_threads.value < 1 << 32, (heads, kv, dim, count, max_kv, most_threads.value)
rope = ops.Rope(ops.rope_config(1024))
for type_ in (ops.TYPE_F32, ops.TYPE_F16):
    for heads in (1, 7, 65536):
        for shift in (0, 4):
            s = ops.rope_heads(A + shift, A + shift, heads, 1024, x_row=1 << 23, x_head=1024)
            rope.apply(type_, s, s, 1 << 23)
            assert most_threads.value < 1 << 32, (type_, heads, shift, most_threads.value)
print("ok")
""")


def test_norm_of_too_many_columns_is_refused(on_host):
    on_host("""
A = 1 << 40
for hidden in ((1 << 30) + 1, (1 << 31) - 1):
    args = ops.norm_args(ops.TYPE_F16, 1, 8, A, d_y=A)
    args.hidden = hidden
    try:
        ops.RmsNorm().run(args)
    except rt.NemoError as e:
        assert "hidden must be" in str(e), e
    else:
        raise AssertionError(hidden)
assert launches.value == 0
print("ok")
""")


def test_a_failed_change_of_attention_keeps_the_one_before(on_host):
    """A second nemo_model_set_attention that fails, wherever it does, frees
    what it allocated itself and not the frequencies that the model has."""
    on_host("""
dims = rt.make_dims(hidden=256, q_heads=4, kv_heads=2, head_dim=64, intermediate=256, layers=2, vocab=300,
                    merge_after_layer=1)
context, model = rt.HipContext.shared(0), ctypes.c_void_p()
_lib.check(L.nemo_model_create(context.ptr, ctypes.byref(dims), ctypes.byref(model)))
last = {k: ctypes.c_void_p.in_dll(host, "host_last_" + k) for k in ("malloc", "free")}

def change(theta):
    return L.nemo_model_set_attention(model, ctypes.byref(ops.model_attention(8, 8, theta=theta)))

assert change(1e4) == 0
kept = last["malloc"].value
failed = 0
while True:
    L.nemo_debug_fail_after(1 + failed)
    status = change(1e5)
    L.nemo_debug_fail_after(0)
    if status == 0:
        break
    failed += 1
    assert last["free"].value != kept, failed
assert failed >= 2 and last["free"].value == kept
print("ok")
""")
