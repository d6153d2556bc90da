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
        return _NBYTES[self]


# Calls build their argument structure and compare sizes in line: a step's smallest launches
# take 3 - 4 us, which a helper call for each buffer would add half of.
_NBYTES = (4, 2, 2, 1)  # of a DType


def _short(what: str, buf, nbytes: int):
    raise InvalidInput(f"{what} holds {buf.nbytes} bytes, {nbytes} are needed")


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
        for name, buf in (("d_k", d_k), ("d_v", d_v)):
            if buf.nbytes < nbytes:
                _short(name, buf, nbytes)
        token, head = (kv_heads * head_dim, head_dim) if layout == "token" else (head_dim, page_size * head_dim)
        self.desc = _native.KvCache(d_k.ptr, d_v.ptr, dtype, kv_heads, head_dim, page_size, n_pages,
                                    page_size * kv_heads * head_dim, token, head, k_scale, v_scale)

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
            if buf.nbytes < nbytes:
                _short(name, buf, nbytes)
            setattr(self, name, buf)
        self._call = lib().openmini_kv_plan

    def run(self, d_cached, d_new, requests: int, d_tables, d_free, n_free: int, d_head=None, stream=None,
            table_stride: int | None = None) -> None:
        """requests' tables grow by the pages that d_new tokens more need, taken from d_free
        (n_free page numbers) at *d_head on (None: at 0)."""
        if requests > self.max_requests:
            raise InvalidInput(f"{requests} requests, planned for {self.max_requests}")
        stride = self.max_pages if table_stride is None else table_stride
        n, table_bytes = 4 * requests, 4 * ((requests - 1) * stride + self.max_pages)
        if d_cached.nbytes < n:
            _short("d_cached", d_cached, n)
        if d_new.nbytes < n:
            _short("d_new", d_new, n)
        if d_free.nbytes < 4 * n_free:
            _short("d_free", d_free, 4 * n_free)
        if d_tables.nbytes < table_bytes:
            _short("d_tables", d_tables, table_bytes)
        rc = self._call(_native.KvPlanArgs(
            d_cached.ptr, d_new.ptr, requests, d_free.ptr, n_free, d_head.ptr if d_head is not None else None, d_tables.ptr, stride,
            self.max_pages, self.page_size, self.max_tokens, self.starts.ptr, self.lens.ptr, self.rows.ptr, self.positions.ptr,
            self.slots.ptr, self.row_lens.ptr, self.counts.ptr), stream)
        if rc:
            check(rc)


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
        self._apply, self._append = lib().openmini_rope_apply, lib().openmini_rope_append

    def apply(self, d_x, x_dtype: DType, d_y, y_dtype: DType, d_positions, tokens: int, heads: int, head_dim: int,
              inverse: bool = False, stream=None, x_stride: int | None = None, y_stride: int | None = None,
              position_stride: int | None = None) -> None:
        """d_y [tokens][heads][head_dim] = d_x turned by the tokens' positions
        (d_positions [axes][tokens]); inverse: turned back, the gradient of x from y's."""
        row = heads * head_dim
        xs, ys = row if x_stride is None else x_stride, row if y_stride is None else y_stride
        ps = tokens if position_stride is None else position_stride
        n = _rows_bytes(tokens, xs, row, _NBYTES[x_dtype])
        if d_x.nbytes < n:
            _short("d_x", d_x, n)
        n = _rows_bytes(tokens, ys, row, _NBYTES[y_dtype])
        if d_y.nbytes < n:
            _short("d_y", d_y, n)
        n = 4 * ((self.n_axes - 1) * ps + tokens)
        if d_positions.nbytes < n:
            _short("d_positions", d_positions, n)
        rc = self._apply(self.handle, _native.RopeArgs(d_x.ptr, d_y.ptr, xs, ys, x_dtype, y_dtype, tokens, heads, head_dim, inverse,
                                                       d_positions.ptr, ps), stream)
        if rc:
            check(rc)

    def append(self, cache: KVCache, d_q, d_k, d_v, in_dtype: DType, d_q_out, q_dtype: DType, d_positions, d_slots, tokens: int,
               q_heads: int, stream=None, q_stride: int | None = None, k_stride: int | None = None,
               v_stride: int | None = None, position_stride: int | None = None) -> None:
        """A step of a layer: d_q_out [tokens][q_heads][head_dim] = q turned; k turned and v
        as it is go to the tokens' slots of the cache (negative: nowhere)."""
        q_row, kv_row = q_heads * cache.head_dim, cache.kv_heads * cache.head_dim
        qs = q_row if q_stride is None else q_stride
        ks, vs = kv_row if k_stride is None else k_stride, kv_row if v_stride is None else v_stride
        ps = tokens if position_stride is None else position_stride
        size = _NBYTES[in_dtype]
        n = _rows_bytes(tokens, qs, q_row, size)
        if d_q.nbytes < n:
            _short("d_q", d_q, n)
        n = _rows_bytes(tokens, ks, kv_row, size)
        if d_k.nbytes < n:
            _short("d_k", d_k, n)
        n = _rows_bytes(tokens, vs, kv_row, size)
        if d_v.nbytes < n:
            _short("d_v", d_v, n)
        n = tokens * q_row * _NBYTES[q_dtype]
        if d_q_out.nbytes < n:
            _short("d_q_out", d_q_out, n)
        n = 4 * ((self.n_axes - 1) * ps + tokens)
        if d_positions.nbytes < n:
            _short("d_positions", d_positions, n)
        if d_slots.nbytes < 4 * tokens:
            _short("d_slots", d_slots, 4 * tokens)
        rc = self._append(self.handle, cache.desc, _native.RopeAppendArgs(
            d_q.ptr, d_k.ptr, d_v.ptr, qs, ks, vs, d_q_out.ptr, q_row, in_dtype, q_dtype, tokens, q_heads, d_positions.ptr, ps,
            d_slots.ptr), stream)
        if rc:
            check(rc)

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
        self._call = lib().openmini_attn_decode

    def run(self, cache: KVCache, d_q, d_out, d_tables, max_pages: int, d_lens, rows: int, d_rows=None,
            requests: int | None = None, d_lse=None, stream=None, table_stride: int | None = None,
            q_stride: int | None = None, out_stride: int | None = None) -> None:
        """d_out [rows][q_heads][head_dim]: row j attends to the first d_lens[j] keys of request
        d_rows[j] (None: of request j), whose pages are d_tables[request][:max_pages];
        d_lse [rows][q_heads] fp32, the log of the sum of exponentials."""
        if cache.kv_heads != self.kv_heads or cache.head_dim != self.head_dim:
            raise InvalidInput(f"cache of {cache.kv_heads} heads of {cache.head_dim}, expected {self.kv_heads} of {self.head_dim}")
        if requests is None:
            if d_rows is not None:
                raise InvalidInput("requests is needed with d_rows")
            requests = rows
        if requests < 1 and rows > 0:
            raise InvalidInput(f"{rows} rows of {requests} requests")
        row = self.q_heads * self.head_dim
        qs, os_ = row if q_stride is None else q_stride, row if out_stride is None else out_stride
        ts = max_pages if table_stride is None else table_stride
        n = _rows_bytes(rows, qs, row, 2)
        if d_q.nbytes < n:
            _short("d_q", d_q, n)
        n = _rows_bytes(rows, os_, row, _NBYTES[self.out_dtype])
        if d_out.nbytes < n:
            _short("d_out", d_out, n)
        n = 4 * rows
        if d_lens.nbytes < n:
            _short("d_lens", d_lens, n)
        if d_rows is not None and d_rows.nbytes < n:
            _short("d_rows", d_rows, n)
        if d_lse is not None and d_lse.nbytes < n * self.q_heads:
            _short("d_lse", d_lse, n * self.q_heads)
        n = 4 * _rows_bytes(requests, ts, max_pages, 1)
        if d_tables.nbytes < n:
            _short("d_tables", d_tables, n)
        rc = self._call(cache.desc, _native.AttnArgs(
            d_q.ptr, qs, d_out.ptr, os_, d_lse.ptr if d_lse is not None else None, self.q_dtype, self.out_dtype, self.q_heads,
            self.scale, self.window, rows, d_lens.ptr, d_rows.ptr if d_rows is not None else None, d_tables.ptr, ts, max_pages,
            max(requests, 1), self.work.ptr, self.work.nbytes), stream)
        if rc:
            check(rc)


__all__ = ["DType", "KVCache", "PagedAttention", "Rope", "StepPlan", "rope_axes", "rope_frequencies"]
