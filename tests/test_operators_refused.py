"""Calls of the attention block's operators that the C ABI refuses, before it
touches a device: every argument is checked first, so a context, a rope and
buffers that are only addresses serve here."""
import ctypes
import math

import pytest

from nemo_amd import _lib
from nemo_amd import operators as ops

FAKE = ctypes.create_string_buffer(256)
AT = (ctypes.addressof(FAKE) + 63) // 64 * 64  # an aligned address


def refused(call, *args, status=1, match=""):
    got = call(*args)
    message = _lib.load().nemo_last_error().decode()
    assert got == status and match in message, (got, message)


@pytest.mark.parametrize("fields,match", [
    (dict(head_dim=63), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(head_dim=2048), "head_dim"),
    (dict(rotary_dim=130), "rotary_dim"), (dict(rotary_dim=7), "rotary_dim"), (dict(rotary_dim=-2), "rotary_dim"),
    (dict(layout=2), "layout"), (dict(scaling=4), "scaling"), (dict(scaling=-1), "scaling"),
    (dict(theta=1.0), "theta"), (dict(theta=math.inf), "theta"), (dict(theta=math.nan), "theta"),
    (dict(scaling=1, factor=0.0), "factor"), (dict(scaling=1, factor=math.nan), "factor"),
    (dict(scaling=2, original_positions=0), "original_positions"),
    (dict(scaling=2, beta_slow=0.0), "beta"), (dict(scaling=2, beta_fast=0.5), "beta"),
    (dict(scaling=3, high_band=1.0), "band"), (dict(scaling=3, low_band=0.0), "band"),
    (dict(magnitude=math.inf), "magnitude"),
])
def test_rope_configurations(fields, match):
    out = ctypes.c_void_p()
    config = ops.rope_config(fields.pop("head_dim", 128), **fields)
    refused(_lib.load().nemo_rope_create, AT, config, ctypes.byref(out), match=match)


def test_rope_calls():
    apply = _lib.load().nemo_rope_apply
    good = ops.rope_heads(AT, AT, 4, 64)
    refused(apply, None, 1, good, None, 1, 0, 0, None, match="null")
    refused(apply, AT, 1, None, None, 1, 0, 0, None, match="null")
    refused(apply, AT, 24, good, None, 1, 0, 0, None, status=5, match="F32, F16 or BF16")
    refused(apply, AT, 1, good, None, -1, 0, 0, None, match="rows")
    refused(apply, AT, 1, good, None, (1 << 23) + 1, 0, 0, None, match="rows")
    refused(apply, AT, 1, ops.rope_heads(0, AT, 4, 64), None, 1, 0, 0, None, match="null")
    refused(apply, AT, 1, good, ops.rope_heads(AT, 0, 4, 64), 1, 0, 0, None, match="null")
    refused(apply, AT, 1, ops.rope_heads(AT, AT + 1, 4, 64), None, 1, 0, 0, None, match="multiple")
    refused(apply, AT, 0, ops.rope_heads(AT + 2, AT, 4, 64), None, 1, 0, 0, None, match="multiple")
    refused(apply, AT, 1, good, ops.rope_heads(AT + 1, AT, 4, 64), 1, 0, 0, None, match="multiple")
    refused(apply, AT, 1, good, None, 1, AT + 4, 0, None, match="multiple")
    refused(apply, AT, 1, ops.rope_heads(AT, AT, -1, 64), None, 1, 0, 0, None, match="heads")
    refused(apply, AT, 1, ops.rope_heads(AT, AT, 4, 64, x_row=-8), None, 1, 0, 0, None, match="strides")
    refused(apply, AT, 1, good, ops.rope_heads(AT, AT, 4, 64, y_head=1 << 24), 1, 0, 0, None, match="strides")


def config(**kw):
    fields = dict(q_heads=8, kv_heads=2, head_dim=64, type_=ops.TYPE_F16, left=10, right=0, sinks=2, scale=0.0)
    return ops.attention_config(**dict(fields, **kw))


BAD_CONFIGS = [
    (dict(q_heads=0), 1, "q_heads"), (dict(kv_heads=0), 1, "q_heads"), (dict(kv_heads=3), 1, "q_heads"),
    (dict(q_heads=2048), 1, "q_heads"), (dict(head_dim=96), 5, "head_dim"), (dict(type_=ops.TYPE_F32), 5, "F16 or BF16"),
    (dict(left=-2), 1, "left"), (dict(right=-2), 1, "left"), (dict(sinks=-1), 1, "sinks"),
    (dict(scale=-1.0), 1, "scale"), (dict(scale=math.nan), 1, "scale"), (dict(scale=math.inf), 1, "scale"),
]


@pytest.mark.parametrize("fields,status,match", BAD_CONFIGS)
def test_attention_configurations(fields, status, match):
    n = ctypes.c_size_t()
    refused(_lib.load().nemo_window_attention_workspace, config(**fields), 1, 1, 1, ctypes.byref(n), status=status,
            match=match)
    refused(_lib.load().nemo_window_attention, AT, config(**fields), ops.AttentionBatch(), None, status=status,
            match=match)


def batch(**kw):
    side = (AT, 512, 64)
    b = ops.attention_batch(1, 1, 1, 1, AT, AT, AT, side, side, side, side)
    for name, value in kw.items():
        setattr(b, name, value)
    return b


@pytest.mark.parametrize("fields,match", [
    (dict(count=-1), "count"), (dict(count=(1 << 20) + 1), "count"), (dict(q_rows=-1), "q_rows"),
    (dict(q_rows=(1 << 23) + 1), "q_rows"), (dict(kv_rows=-1), "kv_rows"), (dict(kv_rows=(1 << 30) + 1), "kv_rows"),
    (dict(max_kv=-1), "max_kv"), (dict(q=None), "null"), (dict(out=None), "null"), (dict(k=None), "null"),
    (dict(v=None), "null"), (dict(q_start=None), "null"), (dict(kv_start=None), "null"), (dict(kv_len=None), "null"),
    (dict(q=AT + 2), "aligned"), (dict(k=AT + 8), "aligned"), (dict(out=AT + 4), "aligned"),
    (dict(q_start=AT + 2), "multiple"), (dict(kv_len=AT + 1), "multiple"), (dict(kv_start=AT + 4), "multiple"),
    (dict(workspace=AT + 1), "aligned"), (dict(q_row=-8), "strides"), (dict(k_row=1 << 24), "strides"),
    (dict(kv_rows=2, k_row=56), "overlap"), (dict(kv_rows=2, v_row=0), "overlap"),
    (dict(v_head=60), "multiples of 8"), (dict(out_row=4), "multiples of 8"),
])
def test_attention_batches(fields, match):
    refused(_lib.load().nemo_window_attention, AT, config(), batch(**fields), None, match=match)


def test_attention_of_too_many_heads():
    refused(_lib.load().nemo_window_attention, AT, config(q_heads=8, kv_heads=8), batch(count=1 << 20), None,
            match="count times kv_heads")


def test_attention_of_nothing_needs_no_buffers():
    run = _lib.load().nemo_window_attention
    assert run(AT, config(), ops.AttentionBatch(), None) == 0
    assert run(AT, config(), batch(q_rows=0, q=None, k=None), None) == 0
    refused(run, None, config(), batch(), None, match="null")
    refused(run, AT, None, batch(), None, match="null")
    refused(run, AT, config(), None, None, match="null")


def norm(**kw):
    args = ops.norm_args(ops.TYPE_F16, 1, 128, AT, AT, 1e-5, d_y8=AT, d_scales=AT)
    for name, value in kw.items():
        setattr(args, name, value)
    return args


@pytest.mark.parametrize("fields,status,match", [
    (dict(type=24), 5, "F32, F16 or BF16"), (dict(hidden=0), 1, "hidden"), (dict(rows=-1), 1, "rows"),
    (dict(rows=(1 << 23) + 1), 1, "rows"), (dict(epsilon=-1.0), 1, "epsilon"), (dict(epsilon=math.nan), 1, "epsilon"),
    (dict(type8=12), 5, "I8 or F8_E4M3"), (dict(group=16), 1, "group"), (dict(group=-32), 1, "group"),
    (dict(hidden=130, group=64), 1, "divide"), (dict(scales=None), 1, "scales"), (dict(x=None), 1, "null"),
    (dict(x=AT + 1), 1, "multiple"), (dict(delta=AT + 1), 1, "multiple"), (dict(y=AT + 3), 1, "multiple"),
    (dict(type=0, x=AT + 2), 1, "multiple"), (dict(weight=AT + 2), 1, "multiple"), (dict(scales=AT + 1), 1, "multiple"),
    (dict(y8=None), 1, "null"), (dict(x_row=-1), 1, "strides"), (dict(y8_row=1 << 24), 1, "strides"),
])
def test_norms(fields, status, match):
    refused(_lib.load().nemo_rmsnorm, AT, norm(**fields), None, status=status, match=match)


def test_norm_of_no_rows():
    assert _lib.load().nemo_rmsnorm(AT, norm(rows=0, x=None), None) == 0
    refused(_lib.load().nemo_rmsnorm, None, norm(), None, match="null")
    refused(_lib.load().nemo_rmsnorm, AT, None, None, match="null")


def test_python_raises():
    with pytest.raises(AttributeError, match="no field"):
        ops.rope_config(64, rotary=32)
    with pytest.raises(_lib.NemoError):
        _lib.check(_lib.load().nemo_rmsnorm(AT, norm(hidden=0), None))
