"""include/openmini_attn.h: its functions are exported and bound one to one, the ctypes and
Rust structures have its fields, and arguments are refused before any device work."""
import ctypes
import os
import re
import shutil
import subprocess

import numpy as np
import pytest

from openmini_qmm import DType, InvalidInput, KVCache, PagedAttention, Rope, _native, rope_axes, rope_frequencies
import attn_ref as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "openmini_attn.h")
FFI = os.path.join(ROOT, "openmini-v1_amd", "rust", "attn_ffi.rs")
STRUCTS = {"openmini_kv_cache_t": _native.KvCache, "openmini_kv_plan_args_t": _native.KvPlanArgs,
           "openmini_rope_args_t": _native.RopeArgs, "openmini_rope_append_args_t": _native.RopeAppendArgs,
           "openmini_attn_args_t": _native.AttnArgs}
C2CT = {"int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "size_t": ctypes.c_size_t, "float": ctypes.c_float}
C2R = {"int": "c_int", "size_t": "usize", "int64_t": "i64", "int32_t": "i32", "float": "f32", "double": "f64", "void": "c_void",
       "openmini_rope_t": "Rope", "openmini_kv_cache_t": "KvCache", "openmini_kv_plan_args_t": "KvPlanArgs",
       "openmini_rope_args_t": "RopeArgs", "openmini_rope_append_args_t": "RopeAppendArgs", "openmini_attn_args_t": "AttnArgs"}


def _text():
    return re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)


def _functions():
    found = re.findall(r"^([\w ]+?[\s\*]+)(openmini_\w+)\s*\(([^;{]*?)\)\s*;", _text(), flags=re.M | re.S)
    return {name: (ret.strip(), [" ".join(p.split()) for p in args.split(",")]) for ret, name, args in found}


def _fields(struct):
    body = re.search(r"typedef struct \{([^{}]*)\}\s*" + struct + ";", _text()).group(1)
    return [(m.group(1).strip(), m.group(2)) for m in re.finditer(r"([\w\s]+?[\s\*]+)(\w+);", body)]


def test_functions_are_exported_and_bound():
    assert sorted(_functions()) == sorted(_native.ATTN_SIGNATURES)
    L = _native.lib()
    for name, (_, params) in _functions().items():
        assert len(getattr(L, name).argtypes) == len(params), name


@pytest.mark.parametrize("name", sorted(STRUCTS))
def test_ctypes_structures_match(name):
    want = [(f, ctypes.c_void_p if "*" in t else C2CT[t.split()[-1]]) for t, f in _fields(name)]
    assert [(f, t) for f, t in STRUCTS[name]._fields_] == want


def _rust_type(t):
    parts = t.split("*")
    r = C2R[[w for w in parts[0].replace("const", " ").split() if w][-1]]
    for level in range(len(parts) - 1):
        r = ("*const " if "const" in parts[level] else "*mut ") + r
    return r


def test_rust_declarations_match():
    src = open(FFI).read()
    block = src[src.index('extern "C" {'):]
    block = block[:block.index("\n}\n")]
    rust = {name: ([p.split(":", 1)[1].strip() for p in args.split(",") if p.strip()], ret.strip() if ret else "void")
            for name, args, ret in re.findall(r"pub fn (openmini_\w+)\((.*?)\)(?:\s*->\s*([^;]+))?;", block, flags=re.S)}
    want = {}
    for name, (ret, params) in _functions().items():
        types = [_rust_type(re.match(r"(.*?)(\w+)$", p).group(1)) for p in params]
        want[name] = (types, "void" if ret == "void" else C2R[ret])
    assert rust == want
    for c_name in STRUCTS:
        body = re.search(r"pub struct " + C2R[c_name] + r" \{(.*?)\}", src, flags=re.S).group(1)
        fields = [(n, t.strip()) for n, t in re.findall(r"pub (\w+): ([^,]+),", body)]
        assert fields == [(f, _rust_type(t) if "*" in t else C2R[t.split()[-1]]) for t, f in _fields(c_name)], c_name


@pytest.mark.skipif(shutil.which("gcc") is None, reason="no C compiler on this machine")
def test_header_is_c(tmp_path):
    f = tmp_path / "a.c"
    f.write_text('#include "openmini_attn.h"\nint main(void) { return sizeof(openmini_attn_args_t) == 0; }\n')
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), "-fsyntax-only", str(f)], check=True)


def _refused(rc, status, word):
    assert rc == status, (rc, _native.last_error())
    assert word in _native.last_error(), _native.last_error()


BAD, NO = _native.ERR_INVALID_PARAM, _native.ERR_UNSUPPORTED
P = 4096  # a pointer that nothing follows: all refusals here precede device work


def _plan_args(**kw):
    a = dict(d_cached=P, d_new=2 * P, requests=2, d_free=3 * P, n_free=4, d_head=None, d_tables=4 * P, table_stride=8, max_pages=8,
             page_size=16, max_tokens=10, d_starts=5 * P, d_lens=6 * P, d_rows=7 * P, d_positions=8 * P, d_slots=9 * P,
             d_row_lens=10 * P, d_counts=11 * P)
    a.update(kw)
    return _native.KvPlanArgs(**a)


@pytest.mark.parametrize("kw,word", [
    (dict(requests=0), "requests"), (dict(requests=4097), "requests"), (dict(page_size=0), "page_size"),
    (dict(max_pages=0), "max_pages"), (dict(max_pages=1 << 28), "max_pages"), (dict(table_stride=7), "table_stride"),
    (dict(max_tokens=0), "max_tokens"), (dict(n_free=-1), "n_free"), (dict(d_cached=None), "d_cached"),
    (dict(d_slots=None), "d_slots"), (dict(d_free=None), "d_free"), (dict(d_new=P + 2), "aligned"),
    (dict(d_lens=P), "one of its inputs"), (dict(d_tables=3 * P), "one of its inputs")])
def test_plan_refusals(kw, word):
    _refused(_native.lib().openmini_kv_plan(_plan_args(**kw), None), BAD, word)


@pytest.mark.parametrize("kw,word", [
    (dict(d_head=11 * P + 12), "d_head and d_counts"), (dict(d_head=6 * P + 4), "d_head and d_lens"),
    (dict(d_cached=5 * P + 8), "d_cached and d_starts"), (dict(d_cached=5 * P - 4), "d_cached and d_starts"),
    (dict(d_new=10 * P + 36), "d_new and d_row_lens"), (dict(d_free=9 * P - 12), "d_free and d_slots"),
    (dict(d_free=4 * P + 60), "d_free and d_tables"), (dict(d_head=4 * P + 4 * 9, table_stride=9), "d_head and d_tables"),
    (dict(d_free=4 * P + 4 * 8, table_stride=9), "d_free and d_tables")])
def test_plan_refuses_overlaps(kw, word):
    """Any element of an output that is one of an input's, not the first alone."""
    _refused(_native.lib().openmini_kv_plan(_plan_args(**kw), None), BAD, word)


@pytest.mark.parametrize("kw", [
    dict(d_head=11 * P + 16), dict(d_head=11 * P - 4), dict(d_head=4 * P + 4 * 8, table_stride=9), dict(d_cached=5 * P + 12),
    dict(d_new=4 * P + 64), dict(d_free=9 * P, n_free=0), dict(d_head=4 * P + 4 * 17, table_stride=9), dict(d_head=None)])
def test_plan_takes_neighbours(kw):
    """Arrays beside each other, a word in the gap after a row of the tables, no list at all: what
    stops the call is that this machine has no GPU."""
    if _native.lib().openmini_qmm_is_available():
        pytest.skip("the pointers are not memory")
    rc = _native.lib().openmini_kv_plan(_plan_args(**kw), None)
    assert rc == _native.ERR_HIP, (rc, _native.last_error())


def test_null_arguments():
    L = _native.lib()
    _refused(L.openmini_kv_plan(None, None), BAD, "null arguments")
    _refused(L.openmini_rope_apply(None, None, None), BAD, "null arguments")
    _refused(L.openmini_rope_apply(None, _native.RopeArgs(), None), BAD, "null rope")
    _refused(L.openmini_rope_append(None, None, None, None), BAD, "null arguments")
    _refused(L.openmini_attn_decode(None, None, None), BAD, "null arguments")
    _refused(L.openmini_attn_decode(None, _native.AttnArgs(), None), BAD, "null cache")
    L.openmini_rope_free(None)


@pytest.mark.parametrize("freq,axis,pairs,axes,scale,word", [
    ([1.0] * 8, None, 2, 1, 1.0, "pairs"), ([1.0] * 8, None, 6, 1, 1.0, "multiple of 4"), ([1.0] * 132, None, 132, 1, 1.0, "pairs"),
    ([1.0] * 8, None, 8, 0, 1.0, "axes"), ([1.0] * 8, None, 8, 9, 1.0, "axes"), ([1.0] * 8, [0] * 7 + [3], 8, 3, 1.0, "axis 3"),
    ([1.0] * 8, [-1] * 8, 8, 3, 1.0, "axis -1"), ([1.0] * 7 + [float("nan")], None, 8, 1, 1.0, "not finite"),
    ([1.0] * 8, None, 8, 1, float("inf"), "not finite"), (None, None, 8, 1, 1.0, "null inv_freq")])
def test_rope_create_refusals(freq, axis, pairs, axes, scale, word):
    f = (ctypes.c_double * len(freq))(*freq) if freq is not None else None
    ax = (ctypes.c_int32 * len(axis))(*axis) if axis is not None else None
    h = ctypes.c_void_p(1)
    _refused(_native.lib().openmini_rope_create(f, ax, pairs, axes, 0, scale, ctypes.byref(h)), BAD, word)
    assert not h.value


def _cache(**kw):
    a = dict(d_k=P, d_v=2 * P, dtype=DType.BF16, kv_heads=2, head_dim=128, page_size=16, n_pages=4, page_stride=4096,
             token_stride=256, head_stride=128, k_scale=1.0, v_scale=1.0)
    a.update(kw)
    return _native.KvCache(**a)


def _attn(**kw):
    a = dict(d_q=P, q_stride=512, d_out=2 * P, out_stride=512, d_lse=None, q_dtype=DType.BF16, out_dtype=DType.F32, q_heads=4,
             scale=0.1, window=0, rows=1, d_lens=3 * P, d_rows=None, d_tables=4 * P, table_stride=4, max_pages=4, requests=1,
             d_work=8 * P, work_bytes=1 << 40)
    a.update(kw)
    return _native.AttnArgs(**a)


@pytest.mark.parametrize("cache,args,status,word", [
    (dict(dtype=0), {}, NO, "cache"), (dict(dtype=4), {}, NO, "cache"), (dict(d_k=None), {}, BAD, "d_k"),
    (dict(d_v=P + 8), {}, BAD, "aligned"), (dict(head_dim=80), {}, NO, "head_dim"), (dict(head_dim=0), {}, BAD, "head_dim"),
    (dict(page_size=12), {}, NO, "page_size"), (dict(page_size=0), {}, BAD, "page_size"), (dict(n_pages=0), {}, BAD, "n_pages"),
    (dict(n_pages=1 << 28), {}, BAD, "n_pages"), (dict(token_stride=12), {}, BAD, "token_stride"),
    (dict(page_stride=-8), {}, BAD, "page_stride"), (dict(k_scale=0.0), {}, BAD, "scales"),
    (dict(v_scale=float("nan")), {}, BAD, "scales"), (dict(kv_heads=0), {}, BAD, "kv_heads"),
    (dict(dtype=DType.F16), {}, NO, "cache of type 1"), ({}, dict(q_dtype=DType.F32), NO, "q"),
    ({}, dict(out_dtype=DType.F16), NO, "out"), ({}, dict(out_dtype=DType.F8_E4M3), NO, "out"), ({}, dict(q_heads=3), BAD, "q_heads"),
    ({}, dict(q_heads=0), BAD, "q_heads"), ({}, dict(rows=-1), BAD, "rows"), ({}, dict(rows=(1 << 20) + 1), BAD, "rows"),
    ({}, dict(d_q=None), BAD, "d_q"), ({}, dict(d_q=P + 2), BAD, "aligned"), ({}, dict(q_stride=504), BAD, "q_stride"),
    ({}, dict(out_stride=514), BAD, "out_stride"), ({}, dict(scale=float("nan")), BAD, "scale"), ({}, dict(window=-1), BAD, "window"),
    ({}, dict(max_pages=0), BAD, "max_pages"), ({}, dict(table_stride=3), BAD, "table_stride"), ({}, dict(requests=0), BAD, "requests"),
    ({}, dict(d_lens=None), BAD, "d_lens"), ({}, dict(d_tables=None), BAD, "d_tables"), ({}, dict(d_work=None), BAD, "d_work"),
    ({}, dict(d_work=8 * P + 128), BAD, "aligned"), ({}, dict(work_bytes=1000), BAD, "workspace"),
    ({}, dict(rows=1 << 20, max_pages=1 << 20, table_stride=1 << 20), BAD, "too many")])
def test_decode_refusals(cache, args, status, word):
    _refused(_native.lib().openmini_attn_decode(_cache(**cache), _attn(**args), None), status, word)


@pytest.mark.parametrize("k_scale,scale", [(1e10, 1e30), (3e38, -2.0), (1.0, 3e38)])
def test_decode_refuses_scales_past_fp32(k_scale, scale):
    """Each finite, their product with log2(e) not: a score of 0 would be NaN."""
    _refused(_native.lib().openmini_attn_decode(_cache(k_scale=k_scale), _attn(scale=scale), None), BAD, "scale")


def test_workspace_bytes():
    L = _native.lib()
    assert L.openmini_attn_workspace_bytes(64, 8, 128) > 0
    for bad in ((0, 0, 128), (4, 0, 128), (4, 3, 128), (4, 8, 128), (4, 4, 100), (2048, 8, 128), (-4, -2, 128)):
        assert L.openmini_attn_workspace_bytes(*bad) == 0, bad


def test_mirror_refusals():
    class Buf:
        ptr, nbytes = ctypes.c_void_p(P), 1000
    with pytest.raises(InvalidInput):
        KVCache(Buf, Buf, DType.BF16, 4, 16, 2, 128)
    with pytest.raises(InvalidInput):
        KVCache(Buf, Buf, DType.BF16, 1, 1, 1, 8, layout="rows")
    with pytest.raises(InvalidInput):
        Rope([1.0] * 8, axes=[0] * 7)
    with pytest.raises(InvalidInput):
        Rope([1.0] * 8, pairing="thirds")
    assert DType.of("f8").nbytes == 1 and DType.of("f32").nbytes == 4


@pytest.mark.parametrize("requests", [0, -1])
def test_rows_need_a_request(requests):
    """Rows that name request 0 of none: the tables' size was not checked for it."""
    class Buf:
        ptr, nbytes = ctypes.c_void_p(P), 1 << 20

    class NoTables:
        ptr, nbytes = ctypes.c_void_p(2 * P), 0
    attn = PagedAttention.__new__(PagedAttention)
    attn.q_heads, attn.kv_heads, attn.head_dim, attn.window, attn.scale = 4, 2, 128, 0, 0.1
    attn.q_dtype, attn.out_dtype, attn.work, attn._call = DType.BF16, DType.F32, Buf, None
    cache = KVCache(Buf, Buf, DType.BF16, 1, 16, 2, 128)
    with pytest.raises(InvalidInput, match="1 rows"):
        attn.run(cache, Buf, Buf, NoTables, 4, Buf, 1, d_rows=Buf, requests=requests)


def test_frequencies_and_axes():
    f = rope_frequencies(64, 500000.0)
    assert len(f) == 64 and f[0] == 1.0 and abs(f[32] - 500000.0 ** -0.5) < 1e-15
    assert rope_axes([2, 1, 3]) == [0, 0, 1, 2, 2, 2]
    assert rope_axes([2, 1, 3], "cycled") == [0, 1, 2, 0, 2, 2]
    with pytest.raises(InvalidInput):
        rope_axes([1], "spiral")


def test_number_formats():
    """The tests' own formats: exact values, ties to even, saturation left to the caller."""
    assert np.array_equal(ref.decode(ref.encode([1.0, -2.5, 448.0, 0.0], ref.F8), ref.F8), [1.0, -2.5, 448.0, 0.0])
    assert ref.decode(ref.encode([17.0, 19.0], ref.F8), ref.F8).tolist() == [16.0, 20.0]
    assert ref.decode(ref.encode([1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8], ref.BF16), ref.BF16).tolist() == [1.0, 1 + 2.0 ** -6]
    assert ref.decode(ref.encode([1 + 2.0 ** -11], ref.F16), ref.F16).tolist() == [1.0]
