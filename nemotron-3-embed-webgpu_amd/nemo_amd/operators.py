"""The attention block's operators on device buffers (include/nemo.h): rotary
positions, alone or behind a norm of each head, attention with a sliding
window and sinks, the residual RMSNorm with 8-bit output, products of such
rows, and a paged cache of 4-bit keys and values with attention over it. With
``QuantWeight.matmul`` they make a layer.

Buffers are device addresses (``tensor.data_ptr()``), strides count elements,
``stream`` is a hipStream_t (0: the default stream); every call enqueues and
returns. The argument structures hold addresses only and may be built once
and passed again for other contents of the same buffers; who keeps one keeps
the buffers too. Nothing here computes.
"""
from __future__ import annotations

import ctypes

from . import _lib
from ._lib import (ROPE_BANDS, ROPE_HALF, ROPE_INTERLEAVED, ROPE_LINEAR, ROPE_NONE, ROPE_YARN, TYPE_BF16, TYPE_F16,
                   TYPE_F32, TYPE_I8, AttentionBatch, AttentionConfig, Cache4Config, Cache4Pages, Cache4Queries,
                   Cache4Rows, HeadNorm, Matmul8Args, ModelAttention, NormArgs, RopeConfig, RopeHeads, check)
from .runtime import HipContext

TYPE_E4M3 = _lib.TYPE_F8_E4M3


def rope_config(head_dim: int, **fields) -> RopeConfig:
    """nemo_rope_config_default with ``head_dim`` and the given fields."""
    c = RopeConfig()
    _lib.load().nemo_rope_config_default(ctypes.byref(c))
    for name, value in dict(fields, head_dim=head_dim).items():
        if not hasattr(c, name):
            raise AttributeError(f"nemo_rope_config has no field {name}")
        setattr(c, name, value)
    return c


def rope_heads(d_x: int, d_y: int, heads: int, head_dim: int, x_row: int | None = None, x_head: int | None = None,
               y_row: int | None = None, y_head: int | None = None) -> RopeHeads:
    """Heads of rows at d_x that go to d_y (the same address: turned in
    place); without strides the rows are ``heads`` dense heads, and those of
    y are those of x."""
    x_head = head_dim if x_head is None else x_head
    x_row = heads * x_head if x_row is None else x_row
    return RopeHeads(d_x, d_y, x_row, x_head, x_row if y_row is None else y_row, x_head if y_head is None else y_head,
                     heads)


def head_norm(d_q_weight: int = 0, d_k_weight: int = 0, epsilon: float = 1e-5, q_weight_head: int = 0,
              k_weight_head: int = 0) -> HeadNorm:
    """Weights [head_dim] of the query and key heads' norms (0: ones); with a
    stride each head has its own."""
    return HeadNorm(d_q_weight, d_k_weight, q_weight_head, k_weight_head, epsilon)


class Rope:
    """Rotary positions of one configuration (nemo_rope)."""

    _ptr = None

    def __init__(self, config: RopeConfig, device: int = 0):
        self.ctx = HipContext.shared(device)
        self.config = config
        ptr = ctypes.c_void_p()
        check(_lib.load().nemo_rope_create(self.ctx.ptr, ctypes.byref(config), ctypes.byref(ptr)))
        self._ptr = ptr
        self._apply = _lib.load().nemo_rope_apply
        self._norm_apply = _lib.load().nemo_rope_norm_apply

    def apply(self, type_: int, q: RopeHeads, k: RopeHeads | None, rows: int, d_positions: int = 0, base: int = 0,
              stream: int = 0) -> None:
        """Turn the heads of ``rows`` tokens; row t has position base +
        positions[t] (int64), or base + t without positions."""
        check(self._apply(self._ptr, type_, q, k, rows, d_positions, base, stream))

    def norm_apply(self, type_: int, q: RopeHeads, k: RopeHeads | None, norm: HeadNorm, rows: int,
                   d_positions: int = 0, base: int = 0, stream: int = 0) -> None:
        """RMSNorm of each head, then ``apply`` of it, in one pass
        (nemo_rope_norm_apply)."""
        check(self._norm_apply(self._ptr, type_, q, k, norm, rows, d_positions, base, stream))

    def destroy(self) -> None:
        ptr, self._ptr = self._ptr, None
        if ptr:
            check(_lib.load().nemo_rope_destroy(ptr))

    def __del__(self):
        try:
            self.destroy()
        except Exception:
            pass


def attention_config(q_heads: int, kv_heads: int, head_dim: int, type_: int = TYPE_F16, left: int = -1,
                     right: int = -1, sinks: int = 0, scale: float = 0.0) -> AttentionConfig:
    """left / right: keys seen before and behind a query (-1: all; right 0 is
    causal); sinks: first keys that stay visible; scale 0: head_dim ** -0.5."""
    return AttentionConfig(q_heads, kv_heads, head_dim, type_, left, right, sinks, scale)


def attention_batch(count: int, q_rows: int, kv_rows: int, max_kv: int, d_q_start: int, d_kv_start: int,
                    d_kv_len: int, q: tuple, k: tuple, v: tuple, out: tuple, d_workspace: int = 0,
                    workspace_bytes: int = 0) -> AttentionBatch:
    """Requests of a batch; q, k, v and out are (address, row stride, head
    stride). The arrays q_start (int32 [count + 1]), kv_start (int64) and
    kv_len (int32) lie on the device. Without a workspace the keys of a query
    are not split over the chip."""
    (dq, q_row, q_head), (dk, k_row, k_head), (dv, v_row, v_head), (do, o_row, o_head) = q, k, v, out
    return AttentionBatch(count, q_rows, kv_rows, max_kv, d_q_start, d_kv_start, d_kv_len, dq, dk, dv, do, q_row,
                          q_head, k_row, k_head, v_row, v_head, o_row, o_head,
                          d_workspace if workspace_bytes else 0, workspace_bytes)


def model_attention(left: int = -1, right: int = -1, sinks: int = 0, global_every: int = 0,
                    **rope_fields) -> ModelAttention:
    """The ``attention`` of a NemotronHipModel: windows and sinks of its
    layers, every ``global_every``-th of which sees all keys, and its rotary
    positions (fields of nemo_rope_config; head_dim is the model's)."""
    return ModelAttention(left, right, sinks, global_every, rope_config(128, **rope_fields))


class WindowAttention:
    """Attention of one configuration (nemo_window_attention)."""

    def __init__(self, config: AttentionConfig, device: int = 0):
        self.ctx = HipContext.shared(device)
        self.config = config
        self._run = _lib.load().nemo_window_attention
        self.workspace_bytes(0, 0, 0)  # the configuration's errors are raised here

    def workspace_bytes(self, count: int, q_rows: int, max_kv: int) -> int:
        n = ctypes.c_size_t(0)
        check(_lib.load().nemo_window_attention_workspace(self.config, count, q_rows, max_kv, ctypes.byref(n)))
        return n.value

    def run(self, batch: AttentionBatch, stream: int = 0) -> None:
        check(self._run(self.ctx.ptr, self.config, batch, stream))


def norm_args(type_: int, rows: int, hidden: int, d_x: int, d_weight: int = 0, epsilon: float = 1e-5,
              d_delta: int = 0, d_sum: int = 0, d_y: int = 0, d_y8: int = 0, type8: int = TYPE_I8, d_scales: int = 0,
              group: int = 0, x_row: int | None = None, delta_row: int | None = None, sum_row: int | None = None,
              y_row: int | None = None, y8_row: int | None = None, scales_row: int | None = None) -> NormArgs:
    """Addresses of 0 are absent; strides that are not given are dense."""
    blocks = hidden // group if group > 0 else 1

    def dense(row):
        return hidden if row is None else row

    return NormArgs(type_, hidden, rows, d_x, d_delta, d_weight, d_sum, d_y, d_y8, d_scales, dense(x_row),
                    dense(delta_row), dense(sum_row), dense(y_row), dense(y8_row),
                    blocks if scales_row is None else scales_row, type8, group, epsilon)


class RmsNorm:
    """Residual addition, RMSNorm and 8-bit output (nemo_rmsnorm)."""

    def __init__(self, device: int = 0):
        self.ctx = HipContext.shared(device)
        self._run = _lib.load().nemo_rmsnorm

    def run(self, args: NormArgs, stream: int = 0) -> None:
        check(self._run(self.ctx.ptr, args, stream))


def matmul8_args(type_: int, m: int, n: int, k: int, d_x: int, d_x_scale: int, d_w: int, d_w_scale: int, d_y: int,
                 d_bias: int = 0, x_row: int | None = None, w_row: int | None = None, y_row: int | None = None,
                 x_scale_row: int = 1) -> Matmul8Args:
    """y [m][n] in ``type_`` of 8-bit rows x [m][k] and weights w [n][k] and
    their float32 scales; rows of x and w begin on 16 bytes, and lie k rounded
    up to 16 apart unless a stride is given."""
    whole = (k + 15) // 16 * 16
    return Matmul8Args(type_, n, k, m, d_x, d_x_scale, d_w, d_w_scale, d_bias, d_y, whole if x_row is None else x_row,
                       x_scale_row, whole if w_row is None else w_row, n if y_row is None else y_row)


class Matmul8:
    """Products of 8-bit rows and weights (nemo_matmul8)."""

    def __init__(self, device: int = 0):
        self.ctx = HipContext.shared(device)
        self._run = _lib.load().nemo_matmul8

    def run(self, args: Matmul8Args, stream: int = 0) -> None:
        check(self._run(self.ctx.ptr, args, stream))


def cache4_config(kv_heads: int, head_dim: int, page: int = 64) -> Cache4Config:
    """A cache of 4-bit keys and values in pages of ``page`` tokens."""
    return Cache4Config(kv_heads, head_dim, page)


def cache4_pages(count: int, pages: int, d_data: int, d_table: int, table_row: int, d_kv_len: int) -> Cache4Pages:
    """Where the tokens of ``count`` requests are: ``pages`` pages at d_data,
    the pages of request b in row b of the table (int32 [count][table_row]),
    kv_len (int32 [count]) tokens each."""
    return Cache4Pages(count, pages, d_data, d_table, table_row, d_kv_len)


def cache4_rows(type_: int, rows: int, d_q_start: int, k: tuple, v: tuple, d_positions: int = 0) -> Cache4Rows:
    """Rows of requests' last tokens; k and v are (address, row stride, head
    stride), q_start (int32 [count + 1]) lies on the device."""
    (dk, k_row, k_head), (dv, v_row, v_head) = k, v
    return Cache4Rows(type_, rows, d_q_start, d_positions, dk, dv, k_row, k_head, v_row, v_head)


def cache4_queries(q_rows: int, max_kv: int, d_q_start: int, q: tuple, out: tuple, d_workspace: int = 0,
                   workspace_bytes: int = 0) -> Cache4Queries:
    """Query rows over a cache; q and out are (address, row stride, head
    stride). Without a workspace the keys of a query are not split over the
    chip."""
    (dq, q_row, q_head), (do, o_row, o_head) = q, out
    return Cache4Queries(q_rows, max_kv, d_q_start, dq, do, q_row, q_head, o_row, o_head,
                         d_workspace if workspace_bytes else 0, workspace_bytes)


class Cache4:
    """A paged cache of 4-bit keys and values (nemo_cache4_*). The pages are
    the caller's: ``page_bytes`` each, and nothing has to be written before
    their tokens are appended."""

    def __init__(self, config: Cache4Config, device: int = 0):
        self.ctx = HipContext.shared(device)
        self.config = config
        n = ctypes.c_size_t(0)
        check(_lib.load().nemo_cache4_page_bytes(config, ctypes.byref(n)))
        self.page_bytes = n.value
        self._append, self._read = _lib.load().nemo_cache4_append, _lib.load().nemo_cache4_read
        self._attention = _lib.load().nemo_cache4_attention

    def append(self, pages: Cache4Pages, rows: Cache4Rows, rope: Rope | None = None, stream: int = 0) -> None:
        """Write the rows of requests' last tokens, keys turned by ``rope``
        (None: as they are)."""
        if rope is not None and not rope._ptr:  # (to the library it would be none)
            raise _lib.NemoError(1, "rope was destroyed")
        check(self._append(self.ctx.ptr, self.config, pages, rows, rope._ptr if rope is not None else None, stream))

    def read(self, pages: Cache4Pages, rows: Cache4Rows, stream: int = 0) -> None:
        """The values of requests' last tokens into rows."""
        check(self._read(self.ctx.ptr, self.config, pages, rows, stream))

    @staticmethod
    def workspace_bytes(attention: AttentionConfig, count: int, q_rows: int, max_kv: int) -> int:
        n = ctypes.c_size_t(0)
        check(_lib.load().nemo_cache4_attention_workspace(attention, count, q_rows, max_kv, ctypes.byref(n)))
        return n.value

    def attention(self, attention: AttentionConfig, pages: Cache4Pages, queries: Cache4Queries, stream: int = 0) -> None:
        """Attention of the query rows over the cache."""
        check(self._attention(self.ctx.ptr, self.config, attention, pages, queries, stream))


__all__ = [
    "ROPE_BANDS", "ROPE_HALF", "ROPE_INTERLEAVED", "ROPE_LINEAR", "ROPE_NONE", "ROPE_YARN", "TYPE_BF16", "TYPE_E4M3",
    "TYPE_F16", "TYPE_F32", "TYPE_I8", "AttentionBatch", "AttentionConfig", "Cache4", "Cache4Config", "Cache4Pages",
    "Cache4Queries", "Cache4Rows", "HeadNorm", "Matmul8", "Matmul8Args", "ModelAttention", "NormArgs", "RmsNorm", "Rope",
    "RopeConfig", "RopeHeads", "WindowAttention", "attention_batch", "attention_config", "cache4_config",
    "cache4_pages", "cache4_queries", "cache4_rows", "head_norm", "matmul8_args", "model_attention", "norm_args",
    "rope_config", "rope_heads",
]
