"""Plain restatements of the attention step in 64 bits, for the tests: number formats,
pages and slots, rotary positions, attention over a paged cache."""
import numpy as np
import torch

F32, F16, BF16, F8 = 0, 1, 2, 3
TORCH = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16, F8: torch.float8_e4m3fn}
BITS = {F32: np.uint32, F16: np.uint16, BF16: np.uint16, F8: np.uint8}
TBITS = {F32: torch.int32, F16: torch.int16, BF16: torch.int16, F8: torch.uint8}
SIZE = {F32: 4, F16: 2, BF16: 2, F8: 1}
# half a unit in the last place of a normal number, relative; half the smallest subnormal
ROUND = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8, F8: 2.0 ** -4}
TINY = {F32: 2.0 ** -150, F16: 2.0 ** -25, BF16: 2.0 ** -134, F8: 2.0 ** -10}


def encode(x, t):
    """float64 / float32 array -> bits of the type, rounded to nearest even."""
    v = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(TORCH[t])
    return v.contiguous().view(TBITS[t]).numpy().view(BITS[t])


def decode(bits, t):
    """Bits of the type -> float64."""
    v = torch.from_numpy(np.ascontiguousarray(bits).view({4: np.int32, 2: np.int16, 1: np.uint8}[SIZE[t]]))
    return v.view(TORCH[t]).float().numpy().astype(np.float64)


def plan(cached, new, free, head, tables, max_pages, page, max_tokens):
    """openmini_kv_plan; `tables` [requests, stride] is changed in place."""
    cached, new = [max(int(c), 0) for c in cached], [max(int(n), 0) for n in new]
    most, R = 2 ** 31 - 1, len(cached)
    out = {k: np.full(max_tokens, -1, np.int32) for k in ("rows", "positions", "slots")}
    out["row_lens"] = np.zeros(max_tokens, np.int32)
    out["starts"], out["lens"] = np.zeros(R + 1, np.int32), np.zeros(R, np.int32)
    head = max(int(head), 0)
    at, used, taken, refused = 0, 0, 0, 0
    for r, (c, n) in enumerate(zip(cached, new)):
        out["starts"][r] = min(at, most)
        held, last = -(-c // page), -(-(c + n) // page)
        too_long = c + n > max_pages * page
        need = 0 if too_long else last - held
        no = too_long or (need > 0 and head + used + need > len(free))
        if not no:
            tables[r, held:held + need] = free[head + used:head + used + need]
            taken += need
        used += need
        refused += no
        out["lens"][r] = c if no else c + n
        for j in range(min(n, max(0, max_tokens - at))):
            p = c + j
            out["rows"][at + j], out["positions"][at + j] = r, min(p, most)
            if not no:
                pg = int(tables[r, p // page])
                s = pg * page + p % page
                out["slots"][at + j] = s if pg >= 0 and s <= most else -1
                out["row_lens"][at + j] = p + 1
        at += n
    out["starts"][R] = min(at, most)
    out["counts"] = np.array([min(at, most), taken, refused, head + taken], np.int32)
    return out


def rope(x, positions, inv_freq, axis, adjacent=False, scale=1.0, inverse=False):
    """x [tokens, heads, dim] float64, positions [axes, tokens]."""
    pairs = len(inv_freq)
    # the angle modulo a turn in integers: positions times revolutions of 2^-80
    turns = [int(round(float(f) / (2 * np.pi) * 2 ** 80)) for f in np.asarray(inv_freq, np.longdouble)]
    frac = np.array([[(int(p) * t) % 2 ** 80 / 2 ** 80 for p in positions[a]] for t, a in zip(turns, axis)]).T
    ang = 2 * np.pi * frac * (-1 if inverse else 1)
    c, s = (np.cos(ang) * scale)[:, None], (np.sin(ang) * scale)[:, None]
    y = np.array(x, np.float64)
    i, j = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if adjacent else (slice(0, pairs), slice(pairs, 2 * pairs))
    a, b = np.array(y[..., i]), np.array(y[..., j])
    y[..., i], y[..., j] = a * c - b * s, a * s + b * c
    return y


def attention(q, keys, values, scale):
    """q [heads, dim], keys and values [n, kv_heads, dim] (only those that are seen), all
    float64: out [heads, dim], lse [heads], and for bounds sum p |v| [heads, dim] and the
    largest |scale| sum |q| |k| [heads]."""
    heads, dim = q.shape
    out, size = np.zeros((heads, dim)), np.zeros((heads, dim))
    lse, dots = np.full(heads, -np.inf), np.zeros(heads)
    if len(keys):
        group = heads // keys.shape[1]
        for h in range(heads):
            k, v = keys[:, h // group], values[:, h // group]
            s = k @ q[h] * scale
            m = s.max()
            p = np.exp(s - m)
            lse[h] = m + np.log(p.sum())
            p /= p.sum()
            out[h], size[h] = p @ v, p @ np.abs(v)
            dots[h] = (np.abs(k) @ np.abs(q[h])).max() * abs(scale)
    return out, lse, size, dots


def attention_bounds(out, size, dots, v_most, dim, q_type, out_type, n):
    """How far the kernel may be off, worst case.  A score: dim products added in 32 bits,
    the scaling, the maximum's difference and the exponential (dim + 16 roundings of
    2^-24 of the sum of magnitudes).  An error e of the scores moves the output by at most
    2 e sum p |v|; the probabilities' two 16-bit parts leave 2^-16 (bf16, 2^-8 of 2^-8) or
    2^-21 (fp16) of each, fp16 subnormals 2^-25 of the largest |v|; sums in 32 bits of n terms,
    32 at a time, and of the waves and parts."""
    e = (dim + 16) * 2.0 ** -24 * dots + 2.0 ** -22
    part = 2.0 ** -16 if q_type == BF16 else 2.0 ** -21
    o = (2 * e[:, None] + part + (n / 32 + 64) * 2.0 ** -24) * size
    if q_type == F16:
        o = o + n * 2.0 ** -25 * v_most
    o = o + ROUND[out_type] * (np.abs(out) + o) + TINY[out_type]
    return o, e + (n / 32 + 64) * 2.0 ** -24 + 2.0 ** -22
