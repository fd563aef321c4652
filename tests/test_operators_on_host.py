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
