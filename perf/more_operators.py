"""The operators of a cache in 8-bit integers with a scale for each block of tokens and head,
and attention of runs of query tokens over a paged cache, one pass each.

A case names an operator and its sizes.  `prepare` makes what a program holds before the
call (the cache, tables, activations and output buffers on the GPU, all values from the
seed; request lengths belong to the case), `run` makes one pass, in elementary torch
operations or, with `own` set, through openmini_qmm; `work` counts the bytes and
operations the result cannot do without; `exact` gives the results in 64 bits from the
operators' definitions.

  write   a step's q turned, k turned and v quantised into their blocks; then the blocks that
          the step touched read back (their codes stand for these values)
  read    the tokens of requests out of the paged cache into dense rows
  decode  attention of one query token a row over an i8 cache
  prompt  attention of runs of query tokens, each seeing the keys up to its own
"""
from __future__ import annotations

import ctypes
import math
import os
import random
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "openmini-v1_amd")
_FLOAT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}
_LEAST_SCALE = 2.0 ** -40
_GROWTH = 1.25  # a block that needs a larger scale takes one this much larger, at least


def _qmm():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import openmini_qmm
    openmini_qmm.init(torch.cuda.current_device())
    return openmini_qmm


def listed():
    return [
        # One conversation's next token through a 70B layer: the smallest write.
        {"name": "write_70b_1", "op": "write", "requests": 1, "least": 1000, "most": 1000, "new": 1, "heads": 64, "kv_heads": 8,
         "dim": 128, "rot": 128, "axes": 1, "pairing": "halves", "in": "f32", "q": "bf16", "block": 16, "page": 16, "layout": "token"},
        # The same for 200 requests decoded together.
        {"name": "write_70b_200", "op": "write", "requests": 200, "least": 30, "most": 4000, "new": 1, "heads": 64, "kv_heads": 8,
         "dim": 128, "rot": 128, "axes": 1, "pairing": "halves", "in": "f32", "q": "bf16", "block": 16, "page": 32, "layout": "token"},
        # A prompt of 8191 tokens behind 9 that are held, images among them, through a 7B layer.
        {"name": "write_7b_8191", "op": "write", "requests": 1, "least": 9, "most": 9, "new": 8191, "heads": 32, "kv_heads": 32,
         "dim": 128, "rot": 128, "axes": 3, "pairing": "halves", "in": "f32", "q": "f16", "block": 32, "page": 64, "layout": "head"},
        # One short conversation read back, as for a move to another server.
        {"name": "read_70b_r1_300", "op": "read", "requests": 1, "least": 300, "most": 300, "first": 0, "kv_heads": 8, "dim": 128,
         "cache": "i8", "block": 16, "page": 16, "layout": "token", "out": "bf16"},
        # Sixty-four ragged requests at once.
        {"name": "read_70b_r64", "op": "read", "requests": 64, "least": 500, "most": 4000, "first": 40, "kv_heads": 8, "dim": 128,
         "cache": "i8", "block": 32, "page": 64, "layout": "head", "out": "f16"},
        # One short conversation, 70B heads: the smallest attention call.
        {"name": "decode_70b_r1_300", "op": "decode", "rows": 1, "least": 300, "most": 300, "heads": 64, "kv_heads": 8, "dim": 128,
         "block": 16, "page": 16, "q": "bf16", "out": "f32", "window": 0, "layout": "token", "empty": 0},
        # One conversation over a long document.
        {"name": "decode_70b_r1_131071", "op": "decode", "rows": 1, "least": 131071, "most": 131071, "heads": 64, "kv_heads": 8,
         "dim": 128, "block": 32, "page": 64, "q": "f16", "out": "f32", "window": 0, "layout": "token", "empty": 0},
        # Sixty-four ragged requests, heads of 64, a sliding window, two rows of padding.
        {"name": "decode_d64_r64_window", "op": "decode", "rows": 64, "least": 50, "most": 16000, "heads": 32, "kv_heads": 4,
         "dim": 64, "block": 8, "page": 16, "q": "bf16", "out": "bf16", "window": 4096, "layout": "head", "empty": 2},
        # A full server on a 70B layer.
        {"name": "decode_70b_r128", "op": "decode", "rows": 128, "least": 2000, "most": 12000, "heads": 64, "kv_heads": 8,
         "dim": 128, "block": 16, "page": 64, "q": "bf16", "out": "bf16", "window": 0, "layout": "token", "empty": 0},
        # A short prompt on a 70B layer.
        {"name": "prompt_70b_211", "op": "prompt", "requests": 1, "least": 0, "most": 0, "new": 211, "short": 211, "heads": 64,
         "kv_heads": 8, "dim": 128, "cache": "i8", "block": 16, "page": 16, "q": "bf16", "out": "bf16", "window": 0, "layout": "token",
         "refused": 0},
        # Pieces of six prompts behind what they hold already, a fp16 cache, output for the fp32 projection; one is refused.
        {"name": "prompt_pieces_f16", "op": "prompt", "requests": 6, "least": 100, "most": 9000, "new": 700, "short": 3, "heads": 32,
         "kv_heads": 8, "dim": 64, "cache": "f16", "block": 0, "page": 16, "q": "f16", "out": "f32", "window": 4096, "layout": "head",
         "refused": 1},
        # A long prompt on a 70B layer: the largest.
        {"name": "prompt_70b_8191", "op": "prompt", "requests": 1, "least": 0, "most": 0, "new": 8191, "short": 8191, "heads": 64,
         "kv_heads": 8, "dim": 128, "cache": "i8", "block": 16, "page": 64, "q": "bf16", "out": "bf16", "window": 0, "layout": "token",
         "refused": 0},
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _pages(rng):
    """A page size and a block that divides it."""
    page = rng.choice([8, 16, 16, 24, 32, 64, 64, 160, 256])
    return {"page": page, "block": rng.choice([b for b in (8, 16, 16, 32) if page % b == 0])}


def _grouped(rng, most=64):
    kv_heads = rng.choice([1, 2, 4, 8, 8, 16, 32])
    return {"kv_heads": kv_heads, "heads": kv_heads * rng.choice([h for h in (1, 2, 3, 4, 5, 7, 8, 16, 32) if kv_heads * h <= most])}


def draw(rng):
    op = rng.choice(["write", "write", "read", "decode", "decode", "decode", "prompt", "prompt", "prompt"])
    dim = rng.choice([64, 96, 128, 128, 128, 192, 256])
    layout = rng.choice(["token", "head"])
    if op == "write":
        c = {"op": op, **_grouped(rng), "dim": dim, "rot": rng.choice([dim, dim, dim // 2]), "axes": rng.choice([1, 1, 3]),
             "pairing": rng.choice(["halves", "halves", "adjacent"]), "in": rng.choice(["f32", "f32", "f16", "bf16"]),
             "q": rng.choice(["bf16", "f16"]), **_pages(rng), "layout": layout}
        tokens = _spread(rng, 1, min(8192, 60000000 // ((c["heads"] + 2 * c["kv_heads"]) * dim)))
        c["requests"] = rng.choice([1, tokens if tokens <= 512 else 3, max(1, min(tokens // 3, 20))])
        c["new"] = max(1, tokens // c["requests"])
        return {**c, "least": 1, "most": _spread(rng, 1, 3000)}
    if op == "read":
        kv_heads, requests = rng.choice([1, 2, 4, 8, 8, 32]), _spread(rng, 1, 200)
        most = _spread(rng, 1, max(1, min(30000, 100000000 // (requests * kv_heads * dim))))
        return {"op": op, "requests": requests, "least": max(1, int(most * rng.choice([1.0, 0.3]))), "most": most,
                "first": rng.choice([0, 0, most // 3]), "kv_heads": kv_heads, "dim": dim, "cache": rng.choice(["i8", "i8", "i8", "f16", "bf16"]),
                **_pages(rng), "layout": layout, "out": rng.choice(["bf16", "f16", "f32"])}
    if op == "decode":
        rows, heads = _spread(rng, 1, 256), _grouped(rng)
        # at most 350M elements of keys, and as many of values, were all rows as long as the longest
        most = _spread(rng, 20, max(21, min(100000, 350000000 // (rows * heads["kv_heads"] * dim))))
        q = rng.choice(["bf16", "f16"])
        return {"op": op, "rows": rows, "least": max(1, int(most * rng.choice([1.0, 0.5, 0.05]))), "most": most, **heads, "dim": dim,
                **_pages(rng), "q": q, "out": rng.choice(["f32", q]), "window": rng.choice([0, 0, 0, 1000]), "layout": layout,
                "empty": min(rows - 1, rng.choice([0, 0, 0, 3]))}
    heads, q, requests = _grouped(rng), rng.choice(["bf16", "f16"]), rng.choice([1, 1, 2, 5, 16])
    new = _spread(rng, 2, 4000 // requests)
    # at most 2^28 pairs of a query token's head and a key, were all requests as long as the longest
    most = rng.choice([0, 0, _spread(rng, 1, max(1, min(20000, (1 << 28) // (requests * new * heads["heads"]))))])
    return {"op": op, "requests": requests, "least": min(1, most), "most": most, "new": new, "short": rng.choice([new, max(1, new // 20)]),
            **heads, "dim": dim, "cache": rng.choice(["i8", "i8", q]), **_pages(rng), "q": q, "out": rng.choice([q, q, "f32"]),
            "window": rng.choice([0, 0, 1000]), "layout": layout, "refused": rng.choice([0, 0, 1]) if requests > 1 else 0}


# ---- inputs ----------------------------------------------------------------------------

class _Dev:
    """A torch tensor as the package's calls take device memory (ptr, nbytes)."""

    def __init__(self, t):
        self.t = t
        self.ptr = ctypes.c_void_p(t.data_ptr())
        self.nbytes = t.numel() * t.element_size()


def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFFFFFF)
    return g


def _normal(g, shape, kind, scale=1.0):
    """N(0, scale) in the type (whole numbers of -127 to 127 in i8), made in pieces so that a
    large cache needs no fp32 copy of itself."""
    out = torch.empty(shape, device="cuda", dtype=_FLOAT[kind])
    flat = out.view(-1)
    for at in range(0, flat.numel(), 1 << 27):
        n = min(1 << 27, flat.numel() - at)
        x = torch.randn(n, generator=g, device="cuda") * scale
        flat[at:at + n] = (x.round().clamp(-127, 127) if kind == "i8" else x).to(_FLOAT[kind])
    return out


def _ints(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def _of_case(case):
    """The random numbers that belong to the case itself, whatever the seed."""
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _lengths(case):
    """For each request of a case: tokens held before the step, tokens of the step (or that are
    read, from the first position on), and the keys that the step's last token sees (0: the
    step refused the request)."""
    rng, op = _of_case(case), case["op"]
    held, new, keys = [], [], []
    for r in range(case["rows"] if op == "decode" else case["requests"]):
        held.append(_spread(rng, case["least"], case["most"]) if case["least"] else 0)
        if op == "decode":
            new.append(1)
            keys.append(case["most"] if r == 0 else held[-1])
        elif op == "read":
            new.append(held[-1] - min(case["first"], held[-1] - 1))
            keys.append(held[-1])
        else:
            new.append(case["new"] if op == "write" or r == 0 else _spread(rng, case["short"], case["new"]))
            keys.append(held[-1] + new[-1])
    for r in rng.sample(range(1, len(keys)), case.get("empty", case.get("refused", 0))):
        keys[r] = 0
    return held, new, keys


def _scale_shape(case, pages):
    each = case["page"] // case["block"]
    return (pages, each, case["kv_heads"]) if case["layout"] == "token" else (pages, case["kv_heads"], each)


def prepare(case, seed):
    st = {"case": case}
    held, new, keys = _lengths(case)
    st["requests"], st["tokens"] = len(held), sum(new)
    _prepare_cache(case, seed, st, held, new, keys)
    {"write": _prepare_write, "read": _prepare_read, "decode": _prepare_decode, "prompt": _prepare_prompt}[case["op"]](
        case, seed, st, held, new, keys)
    if own:
        q = _qmm()
        st["dev"] = {k: _Dev(v) for k, v in st.items() if isinstance(v, torch.Tensor)}
        d, kind = st["dev"], case.get("cache", "i8")
        more = {"block": case["block"], "d_k_scales": d["ks"], "d_v_scales": d["vs"]} if kind == "i8" else {}
        st["cache"] = q.KVCache(d["kc"], d["vc"], q.DType.of(kind), st["pages"], case["page"], case["kv_heads"], case["dim"],
                                layout=case["layout"], **more)
        types = {k: q.DType.of(case[k]) for k in ("in", "q", "out") if k in case}
        st["types"] = types
        if case["op"] == "write":
            st["rope"] = q.Rope(_frequencies(case)[0], axes=_frequencies(case)[1], n_axes=case["axes"], pairing=case["pairing"])
        if case["op"] == "decode":
            st["attn"] = q.PagedAttention(case["heads"], case["kv_heads"], case["dim"], q_dtype=types["q"], out_dtype=types["out"],
                                          window=case["window"])
        if case["op"] == "prompt":
            st["attn"] = q.PromptAttention(case["heads"], case["kv_heads"], case["dim"], q_dtype=types["q"], out_dtype=types["out"],
                                           window=case["window"])
    return st


def _prepare_cache(case, seed, st, held, new, keys):
    """Pages anywhere in the cache, codes over their range and scales that differ from block to block."""
    page, kind = case["page"], case.get("cache", "i8")
    most = [max(k, h + n if case["op"] in ("write", "prompt") else h) for h, n, k in zip(held, new, keys)]
    have = [-(-m // page) for m in most]
    widest = max(max(have), 1)
    pages = sum(have) + 3
    order = torch.randperm(pages, generator=_gen(seed, 1), device="cuda").to(torch.int32)
    count = _ints(have).long()
    before = torch.cumsum(count, 0) - count
    column = torch.arange(widest, device="cuda")[None]
    st["tables"] = torch.where(column < count[:, None], order[(before[:, None] + column).clamp_(max=pages - 1)], 0).contiguous()
    st["pages"], st["widest"] = pages, widest
    shape = (pages, page, case["kv_heads"], case["dim"]) if case["layout"] == "token" else (pages, case["kv_heads"], page, case["dim"])
    for i, name in enumerate(("k", "v")):
        st[name + "c"] = _normal(_gen(seed, 20 + i), shape, kind, 36.0 if kind == "i8" else 1.0)
        if kind == "i8":
            spread = torch.rand(_scale_shape(case, pages), generator=_gen(seed, 30 + i), device="cuda")
            st[name + "s"] = (0.7 + spread) * (3.0 / 127)


def _frequencies(case):
    """Radians a position of each pair, and the pair's axis: the axes in equal blocks of pairs (the first takes the rest)."""
    pairs = case["rot"] // 2
    each = pairs // case["axes"]
    return ([10000.0 ** (-i / pairs) for i in range(pairs)],
            [max(0, i - (pairs - each * case["axes"])) // each for i in range(pairs)])


def _prepare_write(case, seed, st, held, new, keys):
    n, block = st["tokens"], case["block"]
    for i, (name, heads) in enumerate((("q", case["heads"]), ("k", case["kv_heads"]), ("v", case["kv_heads"]))):
        st[name] = _normal(_gen(seed, 10 + i), (n, heads, case["dim"]), case["in"])
    st["held"], st["new"] = _ints(held), _ints(new)
    row = torch.repeat_interleave(torch.arange(len(held), device="cuda"), _ints(new).long(), output_size=n)
    at = torch.arange(n, device="cuda") - (torch.cumsum(st["new"].long(), 0) - st["new"])[row] + st["held"].long()[row]
    st["slots"] = (st["tables"].long()[row, at // case["page"]] * case["page"] + at % case["page"]).int()
    st["pos"] = torch.stack([at] if case["axes"] == 1 else [at // (24 * 42), at // 42 % 24, at % 42]).int().contiguous()
    # the blocks that the step touches, from their first token on
    st["first"] = st["held"] // block * block
    count = st["held"] + st["new"] - st["first"]
    st["starts"] = torch.cat([count.new_zeros(1), torch.cumsum(count, 0).int()])
    st["back"] = sum(h + m - h // block * block for h, m in zip(held, new))
    freq, axis = _frequencies(case)
    st["freq"] = torch.tensor(freq, device="cuda", dtype=torch.float64)
    st["axis"] = torch.tensor(axis, device="cuda", dtype=torch.int64)
    if own:
        st["qo"] = torch.empty(n, case["heads"], case["dim"], device="cuda", dtype=_FLOAT[case["q"]])
        for name in ("ko", "vo"):
            st[name] = torch.empty(st["back"], case["kv_heads"], case["dim"], device="cuda", dtype=_FLOAT[case["q"]])


def _prepare_read(case, seed, st, held, new, keys):
    st["first"] = _ints([h - n for h, n in zip(held, new)])
    st["starts"] = torch.cat([st["first"].new_zeros(1), torch.cumsum(_ints(new), 0).int()])
    if own:
        for name in ("ko", "vo"):
            st[name] = torch.empty(st["tokens"], case["kv_heads"], case["dim"], device="cuda", dtype=_FLOAT[case["out"]])


def _prepare_decode(case, seed, st, held, new, keys):
    st["lens"] = _ints(keys)
    _prepare_queries(case, seed, st)


def _prepare_prompt(case, seed, st, held, new, keys):
    st["starts"] = torch.cat([_ints([0]), torch.cumsum(_ints(new), 0).int()])
    st["longest"] = max(new)
    row = torch.repeat_interleave(torch.arange(len(held), device="cuda"), _ints(new).long(), output_size=st["tokens"])
    last = _ints(keys)[row]  # of the request's last token; each token sees the keys up to its own
    st["lens"] = torch.where(last > 0, torch.arange(st["tokens"], device="cuda") - st["starts"][1:][row] + 1 + last, 0).int()
    _prepare_queries(case, seed, st)


def _prepare_queries(case, seed, st):
    st["q"] = _normal(_gen(seed, 2), (st["tokens"], case["heads"], case["dim"]), case["q"], 1.2)
    if own:
        st["o"] = torch.empty(st["tokens"], case["heads"], case["dim"], device="cuda", dtype=_FLOAT[case["out"]])
        st["lse"] = torch.empty(st["tokens"], case["heads"], device="cuda", dtype=torch.float32)


# ---- one pass --------------------------------------------------------------------------

def run(st):
    op = st["case"]["op"]
    if own:
        return {"write": _own_write, "read": _own_read, "decode": _own_decode, "prompt": _own_prompt}[op](st)
    return {"write": _plain_write, "read": _plain_read, "decode": _plain_decode, "prompt": _plain_prompt}[op](st)


def _own_write(st):
    case, d, types = st["case"], st["dev"], st["types"]
    st["rope"].append(st["cache"], d["q"], d["k"], d["v"], types["in"], d["qo"], types["q"], d["pos"], d["slots"], st["tokens"],
                      case["heads"])
    st["cache"].read(d["tables"], st["widest"], d["starts"], st["requests"], st["back"], d["ko"], d["vo"], types["q"],
                     d_first=d["first"])
    return {"q": st["qo"], "k": st["ko"], "v": st["vo"]}


def _own_read(st):
    d = st["dev"]
    st["cache"].read(d["tables"], st["widest"], d["starts"], st["requests"], st["tokens"], d["ko"], d["vo"], st["types"]["out"],
                     d_first=d["first"])
    return {"k": st["ko"], "v": st["vo"]}


def _own_decode(st):
    d = st["dev"]
    st["attn"].run(st["cache"], d["q"], d["o"], d["tables"], st["widest"], d["lens"], st["tokens"], d_lse=d["lse"])
    return {"o": st["o"], "lse": st["lse"]}


def _own_prompt(st):
    d = st["dev"]
    st["attn"].run(st["cache"], d["q"], d["o"], d["tables"], st["widest"], d["starts"], d["lens"], st["tokens"], st["requests"],
                   d_lse=d["lse"])
    return {"o": st["o"], "lse": st["lse"]}


def _by_token(cache, case):
    """The cache as [pages, page, heads, dim], or its scales as [pages, blocks, heads]."""
    return cache if case["layout"] == "token" else cache.transpose(1, 2)


def _turned(x, st):
    """x [tokens, heads, dim] in 32 bits with its first `rot` dimensions rotated."""
    case, half = st["case"], st["case"]["rot"] // 2
    angle = st["pos"].double()[st["axis"]].t() * st["freq"]  # [tokens, pairs]
    c, s = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    x = x.float()
    turn, rest = x[..., :case["rot"]], x[..., case["rot"]:]
    if case["pairing"] == "halves":
        a, b = turn[..., :half], turn[..., half:]
        return torch.cat([a * c - b * s, a * s + b * c, rest], -1)
    a, b = turn[..., 0::2], turn[..., 1::2]
    return torch.cat([torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2), rest], -1)


def _plain_quantised(x, codes, scales, st):
    """x [tokens, heads, dim] into the blocks of the tokens' slots."""
    case, slots = st["case"], st["slots"].long()
    page, block, n = case["page"], case["block"], x.shape[0]
    codes, scales = _by_token(codes, case), _by_token(scales, case)
    begin = torch.cumsum(st["new"].long(), 0) - st["new"]
    leads = slots % block == 0
    leads[begin] = True
    run_of = torch.cumsum(leads, 0) - 1  # tokens of one block and call
    size = x.abs().amax(-1)
    size = torch.zeros_like(size).scatter_reduce(0, run_of[:, None].expand_as(size), size, "amax")[run_of]
    behind = torch.zeros(n, device="cuda", dtype=torch.int64).scatter_reduce(0, run_of, torch.where(leads, slots % block, 0), "amax")[run_of]
    at, sub = slots // page, slots % page // block
    old = scales[at, sub]
    need = (size * (1.0 / 127)).clamp(min=_LEAST_SCALE)
    new = torch.where((behind == 0)[:, None], need, torch.where(old >= need, old, torch.maximum(need, old * _GROWTH)))
    # what the requests' first blocks hold already
    page0, sub0, hold = at[begin], sub[begin], behind[begin]
    token = sub0[:, None] * block + torch.arange(block, device="cuda")
    was = codes[page0[:, None], token].float()
    by = (old[begin] / new[begin])[:, None, :, None]
    keep = (torch.arange(block, device="cuda") < hold[:, None])[:, :, None, None]
    codes[page0[:, None], token] = torch.where(keep, (was * by).round().clamp(-127, 127), was).to(torch.int8)
    codes[at, slots % page] = (x * (1.0 / new)[..., None]).round().clamp(-127, 127).to(torch.int8)
    scales[at, sub] = new


def _plain_write(st):
    _plain_quantised(_turned(st["k"], st), st["kc"], st["ks"], st)
    _plain_quantised(st["v"].float(), st["vc"], st["vs"], st)
    kind = _FLOAT[st["case"]["q"]]
    k, v = _plain_rows(st, st["back"])
    return {"q": _turned(st["q"], st).to(kind), "k": k.to(kind), "v": v.to(kind)}


def _plain_rows(st, n):
    """The keys and values of the requests' tokens from `first` on, in 32 bits."""
    case, page = st["case"], st["case"]["page"]
    t = torch.arange(n, device="cuda", dtype=torch.int32)
    row = torch.searchsorted(st["starts"][1:].contiguous(), t, right=True)
    at = t - st["starts"][row] + st["first"][row]
    pages, off = st["tables"].long()[row, at // page], (at % page).long()
    k, v = (_by_token(st[c], case)[pages, off].float() for c in ("kc", "vc"))
    if case.get("cache", "i8") != "i8":
        return k, v
    sk, sv = (_by_token(st[c], case)[pages, off // case["block"]][..., None] for c in ("ks", "vs"))
    return k * sk, v * sv


def _plain_read(st):
    k, v = _plain_rows(st, st["tokens"])
    return {"k": k.to(_FLOAT[st["case"]["out"]]), "v": v.to(_FLOAT[st["case"]["out"]])}


def _dense(cache, scales, st):
    """The requests' whole tables in 32 bits: [requests, kv_heads, keys, dim]."""
    case, tables = st["case"], st["tables"].long()
    x = _by_token(cache, case)[tables].float()  # [requests, columns, page, heads, dim]
    if scales is not None:
        r, w, p, h, d = x.shape
        x = (x.view(r, w, p // case["block"], case["block"], h, d) * _by_token(scales, case)[tables][:, :, :, None, :, None]).view(x.shape)
    return x.flatten(1, 2).transpose(1, 2).contiguous()


def _attended(q, lens, st):
    """q [requests, queries, heads, dim], lens [requests, queries]: outputs in 32 bits, laid out as q, and the log of the sums."""
    case = st["case"]
    requests, n, heads, dim = q.shape
    kv_heads = case["kv_heads"]
    group = heads // kv_heads
    k, v = _dense(st["kc"], st.get("ks"), st), _dense(st["vc"], st.get("vs"), st)
    q = q.float().view(requests, n, kv_heads, group, dim).permute(0, 2, 1, 3, 4).reshape(requests, kv_heads, n * group, dim)
    s = torch.matmul(q * (1.0 / math.sqrt(dim)), k.transpose(2, 3).contiguous()).view(requests, kv_heads, n, group, -1)
    j = torch.arange(s.shape[-1], device="cuda")
    seen = j < lens[:, :, None]
    if case["window"]:
        seen = seen & (j >= lens[:, :, None] - case["window"])
    s = s.masked_fill_(~seen[:, None, :, None], -math.inf)
    most = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(most == -math.inf, 0.0, most)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, 1.0, total))
    o = torch.matmul(p.view(requests, kv_heads, n * group, -1), v).view(requests, kv_heads, n, group, dim)
    lse = (most + torch.log(total)).squeeze(-1)
    return o.permute(0, 2, 1, 3, 4).reshape(requests, n, heads, dim), lse.permute(0, 2, 1, 3).reshape(requests, n, heads)


def _plain_decode(st):
    o, lse = _attended(st["q"][:, None], st["lens"].long()[:, None], st)
    return {"o": o[:, 0].to(_FLOAT[st["case"]["out"]]), "lse": lse[:, 0]}


def _plain_prompt(st):
    n, starts = st["longest"], st["starts"].long()
    i = torch.arange(n, device="cuda")
    real = starts[:-1, None] + i < starts[1:, None]
    at = torch.where(real, starts[:-1, None] + i, 0)
    o, lse = _attended(st["q"][at], torch.where(real, st["lens"].long()[at], 0), st)
    # each token's place among the padded ones
    t = torch.arange(st["tokens"], device="cuda")
    row = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    return {"o": o[row, t - starts[row]].to(_FLOAT[st["case"]["out"]]), "lse": lse[row, t - starts[row]]}


# ---- what a pass needs -----------------------------------------------------------------

def work(case):
    held, new, keys = _lengths(case)
    op, d, kv, kind, tokens = case["op"], case["dim"], case["kv_heads"], case.get("cache", "i8"), sum(new)
    block, page, scale_bytes = case["block"], case["page"], 8 * kv  # of a block's keys and values
    if op == "write":
        blocks = sum(-(-(h + n) // block) - h // block for h, n in zip(held, new))
        grown = sum(1 for h in held if h % block)
        back = sum(h + n - h // block * block for h, n in zip(held, new))
        append = tokens * d * ((case["heads"] + 2 * kv) * _SIZE[case["in"]] + case["heads"] * 2 + 2 * kv) + 4 * tokens * (case["axes"] + 1)
        return {"bytes": append + scale_bytes * (2 * blocks + grown) + back * kv * d * 2 * (1 + 2),
                "flops": tokens * (3 * (case["heads"] + kv) * case["rot"] + 2 * kv * d)}
    if op == "read":
        blocks = sum(-(-k // block) - (k - n) // block for k, n in zip(keys, new)) if kind == "i8" else 0
        return {"bytes": 2 * tokens * kv * d * (_SIZE[kind] + _SIZE[case["out"]]) + scale_bytes * blocks + 4 * -(-tokens // page),
                "flops": 0}
    # keys that some query token of a request reads, and pairs of a query token and a key
    read = pairs = 0
    for n, k in zip(new, keys):
        for i in range(n if k else 0):
            pairs += min(k - i, case["window"] or k)
        if k:
            read += min(k, case["window"] + n - 1) if case["window"] else k
    scales = scale_bytes * -(-read // block) if kind == "i8" else 0
    return {"bytes": 2 * read * kv * d * _SIZE[kind] + scales + 4 * -(-read // page) +
            tokens * case["heads"] * (d * (_SIZE[case["q"]] + _SIZE[case["out"]]) + 4) + 4 * tokens, "flops": 4 * pairs * case["heads"] * d}


# ---- the definitions, in 64 bits -------------------------------------------------------

def exact(case, seed):
    """What `run` returns, from the definitions in 64 bits."""
    global own
    was, own = own, False  # the inputs alone
    try:
        st = prepare(case, seed)
    finally:
        own = was
    held, new, keys = _lengths(case)
    if case["op"] == "write":
        return _exact_write(case, st, held, new)
    if case["op"] == "read":
        k, v = zip(*(_exact_keys(case, st, r, torch.arange(end - n, end, device="cuda")) for r, (n, end) in enumerate(zip(new, keys))))
        return {"k": torch.cat(k), "v": torch.cat(v)}
    out = torch.zeros(st["tokens"], case["heads"], case["dim"], device="cuda", dtype=torch.float64)
    lse = torch.full((st["tokens"], case["heads"]), -math.inf, device="cuda", dtype=torch.float64)
    t = 0
    for r, (n, end) in enumerate(zip(new, keys)):
        if end:
            _exact_request(case, st, r, end, slice(t, t + n), out, lse)
        t += n
    return {"o": out, "lse": lse}


def _exact_keys(case, st, r, at):
    """Keys and values of request r at the positions `at`: [n, kv_heads, dim]."""
    page, off = st["tables"][r].long()[at // case["page"]], at % case["page"]
    tokens = case["layout"] == "token"
    both = []
    for name in "kv":
        x = (st[name + "c"][page, off] if tokens else st[name + "c"][page, :, off]).double()
        if name + "s" in st:
            s, b = st[name + "s"], off // case["block"]
            x = x * (s[page, b] if tokens else s[page, :, b]).double()[..., None]
        both.append(x)
    return both


def _exact_request(case, st, r, end, rows, out, lse):
    """The last of the rows sees `end` keys, those before it one less each."""
    n, group = rows.stop - rows.start, case["heads"] // case["kv_heads"]
    lo = max(0, end - n + 1 - case["window"]) if case["window"] else 0
    at = torch.arange(lo, end, device="cuda")
    keys, values = _exact_keys(case, st, r, at)
    last = torch.arange(end - n + 1, end + 1, device="cuda")[:, None]
    hidden = (at >= last) | (at < last - case["window"] if case["window"] else at < 0)
    for h in range(case["heads"]):
        s = (st["q"][rows, h].double() @ keys[:, h // group].t().contiguous() / math.sqrt(case["dim"])).masked_fill_(hidden, -math.inf)
        lse[rows, h] = torch.logsumexp(s, 1)
        out[rows, h] = torch.exp(s.sub_(lse[rows, h, None])) @ values[:, h // group].contiguous()


def _exact_write(case, st, held, new):
    """Each pair as a complex number, times exp(i angle); then request by request, its blocks side by side."""
    freq, axis = _frequencies(case)
    angle = st["pos"].double()[torch.tensor(axis, device="cuda")].t() * torch.tensor(freq, device="cuda", dtype=torch.float64)
    by, half, block = torch.polar(torch.ones_like(angle), angle)[:, None], case["rot"] // 2, case["block"]
    first, second = (slice(0, half), slice(half, 2 * half)) if case["pairing"] == "halves" else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))

    def turn(x):
        y = x.double().clone()
        z = torch.complex(y[..., first], y[..., second]) * by
        y[..., first], y[..., second] = z.real, z.imag
        return y

    out = {"q": turn(st["q"])}
    for i, (name, x) in enumerate((("k", turn(st["k"])), ("v", st["v"].double()))):
        rows, t = [], 0
        for r, (h, n) in enumerate(zip(held, new)):
            start = h // block * block
            behind = h - start
            total = behind + n
            blocks = -(-total // block)
            # the new tokens laid over the touched blocks, zeros elsewhere
            laid = torch.zeros(blocks * block, case["kv_heads"], case["dim"], device="cuda", dtype=torch.float64)
            laid[behind:total] = x[t:t + n]
            laid = laid.view(blocks, block, case["kv_heads"], case["dim"])
            scale = (laid.abs().amax((1, 3)) / 127).clamp(min=_LEAST_SCALE)
            codes = None
            if behind:
                at = st["tables"][r, start // case["page"]].long()
                b, off = start % case["page"] // block, start % case["page"]
                tokens = case["layout"] == "token"
                old = (st[name + "s"][at, b] if tokens else st[name + "s"][at, :, b]).double()
                was = st[name + "c"][at, off:off + behind] if tokens else st[name + "c"][at, :, off:off + behind].transpose(0, 1)
                grown = torch.where(old >= scale[0], old, torch.maximum(scale[0], old * _GROWTH))
                codes = (was.double() * (old / grown)[None, :, None]).round().clamp(-127, 127)
                scale[0] = grown
            c = (laid / scale[:, None, :, None]).round().clamp(-127, 127).view(blocks * block, case["kv_heads"], case["dim"])
            if codes is not None:
                c[:behind] = codes
            rows.append((c.view(laid.shape) * scale[:, None, :, None]).view(c.shape)[:total])
            t += n
        out[name] = torch.cat(rows)
    return out
