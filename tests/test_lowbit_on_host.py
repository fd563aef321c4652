"""Launch sizes of the low-bit operators, on a host whose HIP runtime is
tests/hip_on_host.c."""
import pytest

from test_operators_on_host import on_host  # noqa: F401 (a fixture)


def test_matmul_grids(on_host):  # noqa: F811
    """Every product that is taken, in a grid below 2^32 threads and x of it alone."""
    on_host("""
A = 1 << 40
most = 1 << 23
for m, n in ((1, most), (most, 1), (17, most), (most, 17), (64, most), (1 << 19, 1 << 19), (most, 1 << 15), (1 << 15, most),
             (100003, 70001), (1 << 20, 257), (300, 5000), (1, 1)):
    for k in (0, 1, 128, 2048, 131071):
        for t in (ops.TYPE_F32, ops.TYPE_F16):
            ops.Matmul8().run(ops.matmul8_args(t, m, n, k, A, A, A, A, A, y_row=n, x_row=(k + 15) // 16 * 16))
            assert most_threads.value < 1 << 32, (m, n, k, most_threads.value)
print("ok")
""")


def test_head_norm_grids(on_host):  # noqa: F811
    """(The stand-in counts a grid's first dimension; heads are dealt to its second, at most
    that many as a workgroup's threads leave.)"""
    on_host("""
A = 1 << 40
for dim in (2, 6, 64, 80, 128, 1022, 1024):
    for layout in (ops.ROPE_HALF, ops.ROPE_INTERLEAVED):
        rope = ops.Rope(ops.rope_config(dim, layout=layout))
        for type_ in (ops.TYPE_F32, ops.TYPE_F16):
            for heads in (1, 7, 65536):
                for shift in (0, 4):
                    for rows in (1, 513, 1 << 23):
                        s = ops.rope_heads(A + shift, A + shift, heads, dim, x_row=1 << 23, x_head=dim)
                        rope.norm_apply(type_, s, s, ops.head_norm(), rows)
                        assert most_threads.value < 1 << 32, (dim, type_, heads, shift, rows, most_threads.value)
print("ok")
""")


def test_cache_grids(on_host):  # noqa: F811
    on_host("""
A = 1 << 40
for heads, kv, dim in ((1, 1, 64), (32, 8, 128), (1024, 1, 64), (1024, 1024, 128), (4, 4, 128)):
    cache = ops.Cache4(ops.cache4_config(kv, dim, 1024))
    for count in (1, (1 << 22) // kv if kv >= 4 else 1 << 20):
        pages = ops.cache4_pages(count, 1 << 30, A, A, 1 << 23, A)
        side = (A, heads * dim, dim)
        cache.append(pages, ops.cache4_rows(ops.TYPE_F32, 1 << 23, A, side, side))
        cache.read(pages, ops.cache4_rows(ops.TYPE_F32, 1 << 23, A, side, side))
        assert most_threads.value < 1 << 32
        for max_kv in (1, 1000, 5000, 1 << 30, 1 << 60):
            for rows in (1, 100, (1 << 26) // heads):
                c = ops.attention_config(heads, kv, dim, right=0)
                need = cache.workspace_bytes(c, count, rows, max_kv)
                cache.attention(c, pages, ops.cache4_queries(rows, max_kv, A, side, side, A, need))
                assert most_threads.value < 1 << 32, (heads, kv, dim, count, max_kv, rows, most_threads.value)
print("ok")
""")


def test_a_destroyed_rope_does_not_append_keys_as_they_are(on_host):  # noqa: F811
    """Without a rope keys go in unturned; one that is no longer there is refused, and
    nothing is launched."""
    on_host("""
A = 1 << 40
cache = ops.Cache4(ops.cache4_config(2, 64, 32))
pages = ops.cache4_pages(1, 1, A, A, 1, A)
rows = ops.cache4_rows(ops.TYPE_F16, 1, A, (A, 128, 64), (A, 128, 64))
rope = ops.Rope(ops.rope_config(64))
cache.append(pages, rows, rope)
cache.append(pages, rows)
rope.destroy()
before = launches.value
for call in (lambda: cache.append(pages, rows, rope), lambda: cache.append(pages, rows, rope=rope)):
    try:
        call()
    except rt.NemoError as e:
        assert "destroyed" in str(e), e
    else:
        raise AssertionError("appended")
assert launches.value == before
print("ok")
""")


def test_page_bytes_of_a_cache(on_host):  # noqa: F811
    on_host("""
for heads, dim, page, want in ((1, 64, 32, 32 * 68), (8, 128, 64, 8 * 64 * 136), (1024, 128, 1024, 1024 * 1024 * 136)):
    assert ops.Cache4(ops.cache4_config(heads, dim, page)).page_bytes == want
print("ok")
""")
