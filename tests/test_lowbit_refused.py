"""Calls of the low-bit operators that the C ABI refuses before it touches a
device: contexts, ropes and buffers that are only addresses serve here."""
import ctypes
import math

import pytest

from nemo_amd import _lib
from nemo_amd import operators as ops

FAKE = ctypes.create_string_buffer(4096)  # zeros, also as a context and a rope
AT = (ctypes.addressof(FAKE) + 63) // 64 * 64


def refused(call, *args, status=1, match=""):
    got = call(*args)
    message = _lib.load().nemo_last_error().decode()
    assert got == status and match in message, (got, message)


def test_head_norms():
    run = _lib.load().nemo_rope_norm_apply
    good, norm = ops.rope_heads(AT, AT, 4, 64), ops.head_norm(AT, AT)
    refused(run, None, 1, good, None, norm, 1, 0, 0, None, match="null")
    refused(run, AT, 1, None, None, norm, 1, 0, 0, None, match="null")
    refused(run, AT, 1, good, None, None, 1, 0, 0, None, match="null")
    refused(run, AT, 24, good, None, norm, 1, 0, 0, None, status=5, match="F32, F16 or BF16")
    refused(run, AT, 1, good, None, norm, -1, 0, 0, None, match="rows")
    refused(run, AT, 1, good, None, norm, (1 << 23) + 1, 0, 0, None, match="rows")
    refused(run, AT, 1, ops.rope_heads(0, AT, 4, 64), None, norm, 1, 0, 0, None, match="null")
    refused(run, AT, 1, good, ops.rope_heads(AT + 1, AT, 4, 64), norm, 1, 0, 0, None, match="multiple")
    refused(run, AT, 1, good, None, norm, 1, AT + 4, 0, None, match="multiple")
    refused(run, AT, 1, ops.rope_heads(AT, AT, 4, 64, x_row=-8), None, norm, 1, 0, 0, None, match="strides")
    for bad in (dict(epsilon=-1.0), dict(epsilon=math.nan), dict(epsilon=math.inf)):
        refused(run, AT, 1, good, None, ops.head_norm(AT, AT, **bad), 1, 0, 0, None, match="epsilon")
    refused(run, AT, 1, good, None, ops.head_norm(AT + 2, AT), 1, 0, 0, None, match="multiple")
    refused(run, AT, 1, good, None, ops.head_norm(AT, AT, k_weight_head=-1), 1, 0, 0, None, match="weight strides")


def matmul(**kw):
    args = ops.matmul8_args(ops.TYPE_F16, 2, 3, 32, AT, AT, AT, AT, AT)
    for name, value in kw.items():
        setattr(args, name, value)
    return args


@pytest.mark.parametrize("fields,status,match", [
    (dict(type=24), 5, "F32, F16 or BF16"), (dict(m=-1), 1, "m must"), (dict(m=(1 << 23) + 1), 1, "m must"),
    (dict(n=-1), 1, "n must"), (dict(n=(1 << 23) + 1), 1, "n must"), (dict(m=1 << 23, n=1 << 23), 1, "2^38"),
    (dict(k=-1), 1, "k must"), (dict(k=131072), 1, "k must"), (dict(x=None), 1, "null"), (dict(w=None), 1, "null"),
    (dict(x_scale=None), 1, "null"), (dict(w_scale=None), 1, "null"), (dict(y=None), 1, "null"),
    (dict(x_row=40), 1, "multiples of 16"), (dict(w_row=8), 1, "multiples of 16"), (dict(x_row=16), 1, "overlap"),
    (dict(w_row=0), 1, "overlap"), (dict(y_row=2), 1, "overlap"), (dict(x=AT + 8), 1, "aligned"),
    (dict(w=AT + 4), 1, "aligned"), (dict(y=AT + 1), 1, "multiple"), (dict(type=0, y=AT + 2), 1, "multiple"),
    (dict(bias=AT + 2), 1, "multiple"), (dict(x_scale=AT + 1), 1, "multiple"), (dict(x_row=-16), 1, "strides"),
    (dict(y_row=1 << 24), 1, "strides"), (dict(x_scale_row=-1), 1, "strides"),
])
def test_matmuls(fields, status, match):
    refused(_lib.load().nemo_matmul8, AT, matmul(**fields), None, status=status, match=match)


def test_matmul_of_nothing():
    run = _lib.load().nemo_matmul8
    assert run(AT, matmul(m=0, x=None), None) == 0 and run(AT, matmul(n=0, w=None, y=None), None) == 0
    refused(run, None, matmul(), None, match="null")
    refused(run, AT, None, None, match="null")


BAD_CACHES = [
    (dict(kv_heads=0), 1, "kv_heads"), (dict(kv_heads=1025), 1, "kv_heads"), (dict(head_dim=96), 5, "head_dim"),
    (dict(page=16), 1, "page"), (dict(page=48), 1, "page"), (dict(page=2048), 1, "page"), (dict(page=0), 1, "page"),
]


def cache(**kw):
    return ops.cache4_config(**dict(dict(kv_heads=2, head_dim=64, page=32), **kw))


def pages(**kw):
    p = ops.cache4_pages(1, 1, AT, AT, 1, AT)
    for name, value in kw.items():
        setattr(p, name, value)
    return p


def rows(**kw):
    r = ops.cache4_rows(ops.TYPE_F16, 1, AT, (AT, 128, 64), (AT, 128, 64))
    for name, value in kw.items():
        setattr(r, name, value)
    return r


@pytest.mark.parametrize("fields,status,match", BAD_CACHES)
def test_cache_configurations(fields, status, match):
    L, n = _lib.load(), ctypes.c_size_t()
    refused(L.nemo_cache4_page_bytes, cache(**fields), ctypes.byref(n), status=status, match=match)
    refused(L.nemo_cache4_append, AT, cache(**fields), pages(), rows(), None, None, status=status, match=match)
    refused(L.nemo_cache4_read, AT, cache(**fields), pages(), rows(), None, status=status, match=match)


def test_page_bytes():
    assert ops.Cache4.__init__ is not None
    L, n = _lib.load(), ctypes.c_size_t()
    for heads, dim, page, want in ((1, 64, 32, 32 * 68), (8, 128, 64, 8 * 64 * 136), (1024, 128, 1024, 1024 * 1024 * 136)):
        assert L.nemo_cache4_page_bytes(cache(kv_heads=heads, head_dim=dim, page=page), ctypes.byref(n)) == 0
        assert n.value == want
    refused(L.nemo_cache4_page_bytes, None, ctypes.byref(n), match="null")
    refused(L.nemo_cache4_page_bytes, cache(), None, match="null")


BAD_PAGES = [
    (dict(count=-1), "count"), (dict(count=(1 << 20) + 1), "count"), (dict(pages=-1), "pages"),
    (dict(table_row=-1), "table_row"), (dict(table_row=(1 << 23) + 1), "table_row"), (dict(kv_len=None), "null"),
    (dict(table=None), "null"), (dict(data=None), "null"), (dict(kv_len=AT + 2), "multiple"),
    (dict(table=AT + 1), "multiple"), (dict(data=AT + 8), "aligned"),
]


@pytest.mark.parametrize("fields,match", BAD_PAGES)
def test_cache_pages(fields, match):
    L = _lib.load()
    refused(L.nemo_cache4_append, AT, cache(), pages(**fields), rows(), None, None, match=match)
    refused(L.nemo_cache4_read, AT, cache(), pages(**fields), rows(), None, match=match)
    refused(L.nemo_cache4_attention, AT, cache(), attention(), pages(**fields), queries(), None, match=match)


@pytest.mark.parametrize("fields,status,match", [
    (dict(type=24), 5, "F32, F16 or BF16"), (dict(rows=-1), 1, "rows"), (dict(rows=(1 << 23) + 1), 1, "rows"),
    (dict(q_start=None), 1, "null"), (dict(k=None), 1, "null"), (dict(v=None), 1, "null"), (dict(k=AT + 1), 1, "multiple"),
    (dict(type=0, v=AT + 2), 1, "multiple"), (dict(q_start=AT + 2), 1, "multiple"), (dict(positions=AT + 4), 1, "multiple"),
    (dict(k_row=-1), 1, "strides"), (dict(v_head=1 << 24), 1, "strides"),
])
def test_cache_rows(fields, status, match):
    L = _lib.load()
    refused(L.nemo_cache4_append, AT, cache(), pages(), rows(**fields), None, None, status=status, match=match)
    refused(L.nemo_cache4_read, AT, cache(), pages(), rows(**fields), None, status=status, match=match)


def test_appending_with_another_rope():
    """FAKE as a rope has a head_dim of 0."""
    refused(_lib.load().nemo_cache4_append, AT, cache(), pages(), rows(), AT, None, match="head_dim is not the cache's")


def attention(**kw):
    fields = dict(q_heads=8, kv_heads=2, head_dim=64, type_=ops.TYPE_F16, left=10, right=0, sinks=2, scale=0.0)
    return ops.attention_config(**dict(fields, **kw))


def queries(**kw):
    q = ops.cache4_queries(1, 1, AT, (AT, 512, 64), (AT, 512, 64))
    for name, value in kw.items():
        setattr(q, name, value)
    return q


@pytest.mark.parametrize("fields,status,match", [
    (dict(q_heads=0), 1, "q_heads"), (dict(kv_heads=3), 1, "q_heads"), (dict(head_dim=96), 5, "head_dim"),
    (dict(kv_heads=4), 1, "the cache's"), (dict(head_dim=128), 1, "the cache's"),
    (dict(type_=ops.TYPE_F32), 5, "F16 or BF16"), (dict(left=-2), 1, "left"), (dict(sinks=-1), 1, "sinks"),
    (dict(scale=math.nan), 1, "scale"),
])
def test_attention_configurations(fields, status, match):
    refused(_lib.load().nemo_cache4_attention, AT, cache(), attention(**fields), pages(), queries(), None,
            status=status, match=match)


@pytest.mark.parametrize("fields,match", [
    (dict(q_rows=-1), "q_rows"), (dict(q_rows=(1 << 23) + 1), "q_rows"), (dict(max_kv=-1), "max_kv"),
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(q_start=None), "null"), (dict(q=AT + 8), "aligned"),
    (dict(out=AT + 2), "aligned"), (dict(q_start=AT + 2), "multiple"), (dict(workspace=AT + 8), "aligned"),
    (dict(q_row=60), "multiples of 8"), (dict(out_head=-8), "strides"), (dict(out_row=1 << 24), "strides"),
])
def test_attention_queries(fields, match):
    refused(_lib.load().nemo_cache4_attention, AT, cache(), attention(), pages(), queries(**fields), None, match=match)


def test_attention_workspace():
    L, n = _lib.load(), ctypes.c_size_t()
    assert L.nemo_cache4_attention_workspace(attention(left=-1), 1, 1, 100000, ctypes.byref(n)) == 0 and n.value > 0
    refused(L.nemo_cache4_attention, AT, cache(), attention(left=-1), pages(),
            queries(max_kv=100000, workspace=AT, workspace_bytes=n.value - 1), None, match="workspace has")
    refused(L.nemo_cache4_attention_workspace, attention(), -1, 1, 1, ctypes.byref(n), match="count")
    refused(L.nemo_cache4_attention_workspace, None, 1, 1, 1, ctypes.byref(n), match="null")
    refused(L.nemo_cache4_attention_workspace, attention(), 1, 1, 1, None, match="null")


def test_caches_of_nothing_need_no_buffers():
    L = _lib.load()
    none = pages(count=0, kv_len=None, table=None, data=None)
    empty = rows(rows=0, q_start=None, k=None, v=None)
    for call in (lambda p, r: L.nemo_cache4_append(AT, cache(), p, r, None, None),
                 lambda p, r: L.nemo_cache4_read(AT, cache(), p, r, None)):
        assert call(none, rows()) == 0 and call(pages(), empty) == 0
    assert L.nemo_cache4_attention(AT, cache(), attention(), none, queries(), None) == 0
    assert L.nemo_cache4_attention(AT, cache(), attention(), pages(), queries(q_rows=0, q=None, out=None), None) == 0
    for args in ((None, cache(), pages(), rows()), (AT, None, pages(), rows()), (AT, cache(), None, rows()),
                 (AT, cache(), pages(), None)):
        refused(L.nemo_cache4_append, *args, None, None, match="null")
        refused(L.nemo_cache4_read, *args, None, match="null")
    for args in ((None, cache(), attention(), pages(), queries()), (AT, None, attention(), pages(), queries()),
                 (AT, cache(), None, pages(), queries()), (AT, cache(), attention(), None, queries()),
                 (AT, cache(), attention(), pages(), None)):
        refused(L.nemo_cache4_attention, *args, None, match="null")
