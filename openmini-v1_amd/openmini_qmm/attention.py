"""The attention step between a layer's q / k / v projections and its output projection,
over include/openmini_attn.h:

  StepPlan         pages and slots for a step's tokens, on the GPU (openmini_kv_plan)
  KVCache          one layer's paged keys and values
  Rope             rotary positions with one or more axes: apply() on a dense tensor,
                   append() on a step's q and k with the cache write
  PagedAttention   attention of single query tokens over the cache (openmini_attn_decode)

Buffers are DeviceBuffer or anything with `ptr` (c_void_p) and `nbytes`; calls only enqueue
work on `stream` (None: the null stream).  Sizes that do not fit their buffers raise
InvalidInput; what the library refuses raises QmmError.
"""
from __future__ import annotations

import ctypes
import enum

from . import _native
from ._native import check, lib
from .ops import DeviceBuffer, InvalidInput


class DType(enum.IntEnum):
    """openmini_attn_dtype_t: element types of activations and caches."""
    F32 = 0
    F16 = 1
    BF16 = 2
    F8_E4M3 = 3

    @classmethod
    def of(cls, name: str) -> "DType":
        """From "f32", "f16", "bf16" or "f8"."""
        return {"f32": cls.F32, "f16": cls.F16, "bf16": cls.BF16, "f8": cls.F8_E4M3}[name]

    @property
    def nbytes(self) -> int:
        return (4, 2, 2, 1)[self]


def _need(buf, nbytes: int, what: str):
    """The buffer's pointer, if it holds nbytes."""
    if buf.nbytes < nbytes:
        raise InvalidInput(f"{what} holds {buf.nbytes} bytes, {nbytes} are needed")
    return buf.ptr


def _rows_bytes(rows: int, stride: int, row: int, size: int) -> int:
    return ((rows - 1) * stride + row) * size if rows > 0 else 0


# ---- the cache -------------------------------------------------------------------------

class KVCache:
    """Keys and values of one layer in pages of page_size tokens, in buffers of the caller
    (one type; layout "token": [n_pages][page_size][kv_heads][head_dim], "head":
    [n_pages][kv_heads][page_size][head_dim]).  A stored element stands for itself times
    k_scale (v_scale)."""

    def __init__(self, d_k, d_v, dtype: DType, n_pages: int, page_size: int, kv_heads: int, head_dim: int,
                 layout: str = "token", k_scale: float = 1.0, v_scale: float = 1.0):
        if layout not in ("token", "head"):
            raise InvalidInput(f"layout {layout!r} is neither 'token' nor 'head'")
        dtype = DType(dtype)
        nbytes = n_pages * page_size * kv_heads * head_dim * dtype.nbytes
        self.d_k, self.d_v = d_k, d_v
        self.dtype, self.n_pages, self.page_size = dtype, int(n_pages), int(page_size)
        self.kv_heads, self.head_dim, self.layout = int(kv_heads), int(head_dim), layout
        token, head = (kv_heads * head_dim, head_dim) if layout == "token" else (head_dim, page_size * head_dim)
        self.desc = _native.KvCache(_need(d_k, nbytes, "d_k"), _need(d_v, nbytes, "d_v"), dtype, kv_heads, head_dim, page_size,
                                    n_pages, page_size * kv_heads * head_dim, token, head, k_scale, v_scale)

    @classmethod
    def allocate(cls, dtype: DType, n_pages: int, page_size: int, kv_heads: int, head_dim: int, **kw) -> "KVCache":
        nbytes = n_pages * page_size * kv_heads * head_dim * DType(dtype).nbytes
        return cls(DeviceBuffer(nbytes), DeviceBuffer(nbytes), dtype, n_pages, page_size, kv_heads, head_dim, **kw)


# ---- pages and slots -------------------------------------------------------------------

class StepPlan:
    """Pages and slots of a step's tokens (openmini_kv_plan), for steps of up to
    max_requests requests and max_tokens tokens over tables of max_pages columns.  Outputs,
    int32 on the device: starts [requests + 1], lens [requests], counts [4] and, for each
    token, rows, positions, slots and row_lens [max_tokens]; `buffers` may name buffers for
    some of them."""

    _OUT = ("starts", "lens", "rows", "positions", "slots", "row_lens", "counts")

    def __init__(self, page_size: int, max_requests: int, max_tokens: int, max_pages: int, buffers: dict | None = None):
        self.page_size, self.max_requests = int(page_size), int(max_requests)
        self.max_tokens, self.max_pages = int(max_tokens), int(max_pages)
        unknown = set(buffers or ()) - set(self._OUT)
        if unknown:
            raise InvalidInput(f"unknown outputs {sorted(unknown)}")
        sizes = {"starts": max_requests + 1, "lens": max_requests, "counts": 4}
        for name in self._OUT:
            nbytes = 4 * sizes.get(name, max_tokens)
            buf = (buffers or {}).get(name)
            if buf is None:
                buf = DeviceBuffer(nbytes)
            _need(buf, nbytes, name)
            setattr(self, name, buf)

    def run(self, d_cached, d_new, requests: int, d_tables, d_free, n_free: int, d_head=None, stream=None,
            table_stride: int | None = None) -> None:
        """requests' tables grow by the pages that d_new tokens more need, taken from d_free
        (n_free page numbers) at *d_head on (None: at 0)."""
        if requests > self.max_requests:
            raise InvalidInput(f"{requests} requests, planned for {self.max_requests}")
        stride = self.max_pages if table_stride is None else table_stride
        a = _native.KvPlanArgs(_need(d_cached, 4 * requests, "d_cached"), _need(d_new, 4 * requests, "d_new"), requests,
                               _need(d_free, 4 * n_free, "d_free"), n_free, d_head.ptr if d_head is not None else None,
                               _need(d_tables, 4 * _rows_bytes(requests, stride, self.max_pages, 1), "d_tables"), stride,
                               self.max_pages, self.page_size, self.max_tokens, self.starts.ptr, self.lens.ptr, self.rows.ptr,
                               self.positions.ptr, self.slots.ptr, self.row_lens.ptr, self.counts.ptr)
        check(lib().openmini_kv_plan(a, stream))


# ---- rotary positions ------------------------------------------------------------------

def rope_frequencies(pairs: int, base: float = 10000.0) -> list:
    """base^(-i / pairs) radians a position for pair i."""
    return [float(base) ** (-i / pairs) for i in range(pairs)]


def rope_axes(sections, order: str = "blocks") -> list:
    """The axis of each pair: sections[a] pairs for axis a, in blocks one after the other or
    (order "cycled") the axes in turn for as long as each has pairs left."""
    if order == "blocks":
        return [a for a, n in enumerate(sections) for _ in range(n)]
    if order != "cycled":
        raise InvalidInput(f"order {order!r} is neither 'blocks' nor 'cycled'")
    left, out = list(sections), []
    while any(left):
        for a, n in enumerate(left):
            if n:
                left[a] -= 1
                out.append(a)
    return out


class Rope:
    """Rotary positions: pair i of a head turns by position[axes[i]] * inv_freq[i] radians
    (openmini_rope_create).  `pairing`: "halves", dimensions (i, i + pairs), or "adjacent",
    (2 i, 2 i + 1).  `scale` multiplies what is turned."""

    def __init__(self, inv_freq, axes=None, n_axes: int | None = None, pairing: str = "halves", scale: float = 1.0):
        if pairing not in ("halves", "adjacent"):
            raise InvalidInput(f"pairing {pairing!r} is neither 'halves' nor 'adjacent'")
        self.pairs = len(inv_freq)
        if axes is not None and len(axes) != self.pairs:
            raise InvalidInput(f"{len(axes)} axes for {self.pairs} pairs")
        self.n_axes = int(n_axes) if n_axes is not None else (max(axes) + 1 if axes is not None and len(axes) else 1)
        freq = (ctypes.c_double * max(self.pairs, 1))(*inv_freq)
        axis = (ctypes.c_int32 * self.pairs)(*axes) if axes is not None else None
        self.handle = ctypes.c_void_p()
        check(lib().openmini_rope_create(freq, axis, self.pairs, self.n_axes, int(pairing == "adjacent"), scale,
                                         ctypes.byref(self.handle)))

    def _positions(self, d_positions, position_stride, tokens: int):
        stride = tokens if position_stride is None else position_stride
        return _need(d_positions, 4 * _rows_bytes(self.n_axes if tokens else 0, stride, tokens, 1), "d_positions"), stride

    def apply(self, d_x, x_dtype: DType, d_y, y_dtype: DType, d_positions, tokens: int, heads: int, head_dim: int,
              inverse: bool = False, stream=None, x_stride: int | None = None, y_stride: int | None = None,
              position_stride: int | None = None) -> None:
        """d_y [tokens][heads][head_dim] = d_x turned by the tokens' positions
        (d_positions [axes][tokens]); inverse: turned back, the gradient of x from y's."""
        row = heads * head_dim
        xs, ys = row if x_stride is None else x_stride, row if y_stride is None else y_stride
        pos, ps = self._positions(d_positions, position_stride, tokens)
        a = _native.RopeArgs(_need(d_x, _rows_bytes(tokens, xs, row, DType(x_dtype).nbytes), "d_x"),
                             _need(d_y, _rows_bytes(tokens, ys, row, DType(y_dtype).nbytes), "d_y"), xs, ys, x_dtype, y_dtype,
                             tokens, heads, head_dim, bool(inverse), pos, ps)
        check(lib().openmini_rope_apply(self.handle, a, stream))

    def append(self, cache: KVCache, d_q, d_k, d_v, in_dtype: DType, d_q_out, q_dtype: DType, d_positions, d_slots, tokens: int,
               q_heads: int, stream=None, q_stride: int | None = None, k_stride: int | None = None,
               v_stride: int | None = None, position_stride: int | None = None) -> None:
        """A step of a layer: d_q_out [tokens][q_heads][head_dim] = q turned; k turned and v
        as it is go to the tokens' slots of the cache (negative: nowhere)."""
        q_row, kv_row = q_heads * cache.head_dim, cache.kv_heads * cache.head_dim
        qs = q_row if q_stride is None else q_stride
        ks, vs = kv_row if k_stride is None else k_stride, kv_row if v_stride is None else v_stride
        size = DType(in_dtype).nbytes
        pos, ps = self._positions(d_positions, position_stride, tokens)
        a = _native.RopeAppendArgs(_need(d_q, _rows_bytes(tokens, qs, q_row, size), "d_q"),
                                   _need(d_k, _rows_bytes(tokens, ks, kv_row, size), "d_k"),
                                   _need(d_v, _rows_bytes(tokens, vs, kv_row, size), "d_v"), qs, ks, vs,
                                   _need(d_q_out, tokens * q_row * DType(q_dtype).nbytes, "d_q_out"), q_row, in_dtype, q_dtype,
                                   tokens, q_heads, pos, ps, _need(d_slots, 4 * tokens, "d_slots"))
        check(lib().openmini_rope_append(self.handle, cache.desc, a, stream))

    def close(self) -> None:
        if self.handle:
            lib().openmini_rope_free(self.handle)
            self.handle = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ---- attention -------------------------------------------------------------------------

class PagedAttention:
    """Attention of single query tokens over a paged cache (openmini_attn_decode), with the
    workspace that its calls take turns with: one object for calls that follow each other.
    scale None: 1 / sqrt(head_dim).  window > 0: each row sees its last `window` keys."""

    def __init__(self, q_heads: int, kv_heads: int, head_dim: int, q_dtype: DType = DType.BF16, out_dtype: DType = DType.F32,
                 scale: float | None = None, window: int = 0):
        self.q_heads, self.kv_heads, self.head_dim = int(q_heads), int(kv_heads), int(head_dim)
        self.q_dtype, self.out_dtype = DType(q_dtype), DType(out_dtype)
        self.scale = self.head_dim ** -0.5 if scale is None else float(scale)
        self.window = int(window)
        nbytes = lib().openmini_attn_workspace_bytes(self.q_heads, self.kv_heads, self.head_dim)
        if not nbytes:
            raise InvalidInput(f"no attention of {q_heads} query heads on {kv_heads} key heads of {head_dim}")
        self.work = DeviceBuffer(nbytes)
        self.work.fill(0)
        check(lib().openmini_qmm_stream_synchronize(None))  # before a call on any stream

    def run(self, cache: KVCache, d_q, d_out, d_tables, max_pages: int, d_lens, rows: int, d_rows=None,
            requests: int | None = None, d_lse=None, stream=None, table_stride: int | None = None,
            q_stride: int | None = None, out_stride: int | None = None) -> None:
        """d_out [rows][q_heads][head_dim]: row j attends to the first d_lens[j] keys of request
        d_rows[j] (None: of request j), whose pages are d_tables[request][:max_pages];
        d_lse [rows][q_heads] fp32, the log of the sum of exponentials."""
        if (cache.kv_heads, cache.head_dim) != (self.kv_heads, self.head_dim):
            raise InvalidInput(f"cache of {cache.kv_heads} heads of {cache.head_dim}, expected {self.kv_heads} of {self.head_dim}")
        if requests is None:
            if d_rows is not None:
                raise InvalidInput("requests is needed with d_rows")
            requests = rows
        row = self.q_heads * self.head_dim
        qs, os_ = row if q_stride is None else q_stride, row if out_stride is None else out_stride
        ts = max_pages if table_stride is None else table_stride
        a = _native.AttnArgs(_need(d_q, _rows_bytes(rows, qs, row, 2), "d_q"), qs,
                             _need(d_out, _rows_bytes(rows, os_, row, self.out_dtype.nbytes), "d_out"), os_,
                             _need(d_lse, 4 * rows * self.q_heads, "d_lse") if d_lse is not None else None, self.q_dtype,
                             self.out_dtype, self.q_heads, self.scale, self.window, rows, _need(d_lens, 4 * rows, "d_lens"),
                             _need(d_rows, 4 * rows, "d_rows") if d_rows is not None else None,
                             _need(d_tables, 4 * _rows_bytes(requests, ts, max_pages, 1), "d_tables"), ts, max_pages,
                             max(requests, 1), self.work.ptr, self.work.nbytes)
        check(lib().openmini_attn_decode(cache.desc, a, stream))


__all__ = ["DType", "KVCache", "PagedAttention", "Rope", "StepPlan", "rope_axes", "rope_frequencies"]
