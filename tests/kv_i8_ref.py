"""Plain restatements for caches of 8-bit integers, and paged caches of every type for the tests
of what reads them."""
import ctypes

import numpy as np

import attn_ref as ref
from attn_ref import BF16, F16, F32, F8

I8 = 4
SIZE = {**ref.SIZE, I8: 1}
BITS = {**ref.BITS, I8: np.int8}
NAN = {BF16: 0x7FC0, F16: 0x7E00, F8: 0x7F}
f32 = np.float32


def runs(slots, block, n_slots):
    """[(first token, count)]: tokens one behind the other whose slots are one apart, in one block."""
    out = []
    for j, s in enumerate(slots):
        if not 0 <= s < n_slots:
            continue
        if out and sum(out[-1]) == j and s == slots[j - 1] + 1 and s % block:
            out[-1][1] += 1
        else:
            out.append([j, 1])
    return [tuple(r) for r in out]


def new_scale(most, held, old):
    """In 32 bits throughout, as the header has it: the kernel's must be the same for equal `most`."""
    if not np.isfinite(most):
        return f32(np.nan)
    need = max(f32(most) * f32(1.0 / 127), f32(2.0 ** -40))
    if not held:
        return need
    return max(need, f32(old) * f32(1.25)) if old < need else f32(old)


def codes_of(x, scale):
    return np.clip(np.rint(x.astype(np.float32) * (f32(1) / f32(scale))), -127, 127).astype(np.int8)


def rescaled(codes, old, scale):
    return np.clip(np.rint(codes.astype(np.float32) * (f32(old) / f32(scale))), -127, 127).astype(np.int8)


class Paged:
    """Requests of `lens` tokens in pages anywhere in a cache of type c_t (layout "token" or "head").
    What no request holds is NaN, in I8 codes of 127 under scales of NaN; table entries past a
    request's pages are anything at all.  keys[r], values[r] [n, kv, dim] in 64 bits."""

    def __init__(self, qmm, lens, kv, dim, c_t, page=16, block=16, layout="token", seed=0, k_size=1.0, max_pages=None, extra=3):
        self.rng = rng = np.random.default_rng(seed)
        self.lens, self.kv, self.dim, self.c_t, self.page, self.block, self.layout = list(lens), kv, dim, c_t, page, block, layout
        held = [-(-n // page) for n in lens]
        self.max_pages = max_pages or max(max(held), 1)
        self.n_pages = sum(held) + extra
        order = rng.permutation(self.n_pages).astype(np.int32)
        self.tables = rng.choice(np.array([-1, -2 ** 31, 2 ** 31 - 1, self.n_pages, 0], np.int32), (len(lens), self.max_pages))
        at = 0
        for r, h in enumerate(held):
            self.tables[r, :h] = order[at:at + h]
            at += h
        self.k_scale, self.v_scale = (0.0625, 0.3) if c_t == F8 else (1.0, 1.0)
        shape = (self.n_pages, page, kv, dim)
        self.bits = [np.full(shape, 127 if c_t == I8 else NAN[c_t], BITS[c_t]) for _ in range(2)]
        self.scales = [np.full((self.n_pages, page // block, kv), np.nan, np.float32) for _ in range(2)] if c_t == I8 else None
        for r, n in enumerate(lens):
            if n == 0:
                continue
            pg, off = self.tables[r][np.arange(n) // page], np.arange(n) % page
            for i, size in enumerate((k_size, 1.0)):
                if c_t == I8:
                    self.bits[i][pg, off] = np.clip(np.rint(rng.standard_normal((n, kv, dim)) * 40), -127, 127)
                    self.scales[i][pg, off // block] = (size * np.exp(rng.uniform(-5.5, -2.5, (n, kv)))).astype(np.float32)
                else:
                    spread = 16.0 if c_t == F8 else 1.0
                    self.bits[i][pg, off] = ref.encode(rng.standard_normal((n, kv, dim)) * size * spread, c_t)
        self.upload(qmm)

    def element(self, i, pages, offs):
        """Keys (i = 0) or values (1) at these places, in 64 bits."""
        b = self.bits[i][pages, offs]
        if self.c_t != I8:
            return ref.decode(b, self.c_t) * float(np.float32((self.k_scale, self.v_scale)[i]))
        return b.astype(np.float64) * self.scales[i][pages, offs // self.block].astype(np.float64)[..., None]

    def tokens(self, r, at):
        at = np.asarray(at, np.int64)
        pages = self.tables[r][at // self.page]
        pages = np.where((pages >= 0) & (pages < self.n_pages), pages, 0)  # hidden from every row, whatever is there
        return self.element(0, pages, at % self.page), self.element(1, pages, at % self.page)

    def laid(self, a):
        return np.ascontiguousarray(a if self.layout == "token" else a.swapaxes(1, 2))

    def upload(self, qmm):
        buf = qmm.DeviceBuffer.from_numpy
        self.d_k, self.d_v = (buf(self.laid(b)) for b in self.bits)
        more = {}
        if self.c_t == I8:
            self.d_ks, self.d_vs = (buf(self.laid(s)) for s in self.scales)
            more = dict(block=self.block, d_k_scales=self.d_ks, d_v_scales=self.d_vs)
        self.d_tables = buf(self.tables)
        self.cache = qmm.KVCache(self.d_k, self.d_v, self.c_t, self.n_pages, self.page, self.kv, self.dim, layout=self.layout,
                                 k_scale=self.k_scale, v_scale=self.v_scale, **more)

    def download(self, stream=None):
        """(codes, scales) of keys and of values as they are on the device now."""
        def back(d, like):
            shape = self.laid(like).shape
            return self.laid(d.download(like.dtype, shape, stream))
        return [(back(d, b), back(s, sc)) for d, b, s, sc in zip((self.d_k, self.d_v), self.bits, (self.d_ks, self.d_vs), self.scales)]


def at_page(buf, offset, nbytes):
    """Part of a buffer, as calls take one."""
    return type("At", (), dict(ptr=ctypes.c_void_p(buf.ptr.value + offset), nbytes=nbytes))
