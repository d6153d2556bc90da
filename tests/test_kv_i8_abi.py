"""include/openmini_kv_i8.h: its functions are exported and bound one to one, the ctypes and
Rust structures have its fields, and arguments are refused before any device work."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest

from openmini_qmm import DType, InvalidInput, KVCache, PromptAttention, _native
from test_attn_abi import BAD, NO, P, _refused

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "openmini_kv_i8.h")
FFI = os.path.join(ROOT, "openmini-v1_amd", "rust", "kv_i8_ffi.rs")
STRUCTS = {"openmini_kv_scales_t": _native.KvScales, "openmini_kv_read_args_t": _native.KvReadArgs,
           "openmini_attn_prompt_args_t": _native.PromptArgs}
C2CT = {"int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "size_t": ctypes.c_size_t, "float": ctypes.c_float}
C2R = {"int": "c_int", "size_t": "usize", "int64_t": "i64", "int32_t": "i32", "float": "f32", "void": "c_void", "openmini_rope_t": "Rope",
       "openmini_kv_cache_t": "KvCache", "openmini_kv_scales_t": "KvScales", "openmini_kv_read_args_t": "KvReadArgs",
       "openmini_rope_append_args_t": "RopeAppendArgs", "openmini_attn_args_t": "AttnArgs", "openmini_attn_prompt_args_t": "PromptArgs"}


def _text():
    return re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)


def _functions():
    found = re.findall(r"^([\w ]+?[\s\*]+)(openmini_\w+)\s*\(([^;{]*?)\)\s*;", _text(), flags=re.M | re.S)
    return {name: (ret.strip(), [" ".join(p.split()) for p in args.split(",")]) for ret, name, args in found}


def _fields(struct):
    body = re.search(r"typedef struct \{([^{}]*)\}\s*" + struct + ";", _text()).group(1)
    return [(m.group(1).strip(), m.group(2)) for m in re.finditer(r"([\w\s]+?[\s\*]+)(\w+);", body)]


def _rust_type(t):
    parts = t.split("*")
    r = C2R[[w for w in parts[0].replace("const", " ").split() if w][-1]]
    for level in range(len(parts) - 1):
        r = ("*const " if "const" in parts[level] else "*mut ") + r
    return r


def test_functions_are_exported_and_bound():
    assert sorted(_functions()) == sorted(_native.KV_I8_SIGNATURES) and len(_functions()) == 5
    for name, (_, params) in _functions().items():
        assert len(getattr(_native.lib(), name).argtypes) == len(params), name


@pytest.mark.parametrize("name", sorted(STRUCTS))
def test_structures_match(name):
    want = [(f, ctypes.c_void_p if "*" in t else C2CT[t.split()[-1]]) for t, f in _fields(name)]
    assert [(f, t) for f, t in STRUCTS[name]._fields_] == want
    body = re.search(r"pub struct " + C2R[name] + r" \{(.*?)\}", open(FFI).read(), flags=re.S).group(1)
    fields = [(n, t.strip()) for n, t in re.findall(r"pub (\w+): ([^,]+),", body)]
    assert fields == [(f, _rust_type(t) if "*" in t else C2R[t.split()[-1]]) for t, f in _fields(name)]


def test_rust_functions_match():
    src = open(FFI).read()
    block = src[src.index('extern "C" {'):]
    rust = {name: ([p.split(":", 1)[1].strip() for p in args.split(",") if p.strip()], ret.strip() if ret else "void")
            for name, args, ret in re.findall(r"pub fn (openmini_\w+)\((.*?)\)(?:\s*->\s*([^;]+))?;", block, flags=re.S)}
    assert rust == {name: ([_rust_type(re.match(r"(.*?)(\w+)$", p).group(1)) for p in params], C2R[ret])
                    for name, (ret, params) in _functions().items()}
    assert re.search(r"#define OPENMINI_ATTN_I8 (\d+)", _text()).group(1) == re.search(r"pub const I8: i32 = (\d+);", src).group(1) == \
        str(int(DType.I8))


@pytest.mark.skipif(shutil.which("gcc") is None, reason="no C compiler on this machine")
def test_header_is_c(tmp_path):
    f = tmp_path / "a.c"
    f.write_text('#include "openmini_kv_i8.h"\nint main(void) { return sizeof(openmini_attn_prompt_args_t) == 0; }\n')
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), "-fsyntax-only", str(f)], check=True)


def _cache(**kw):
    a = dict(d_k=P, d_v=2 * P, dtype=DType.I8, kv_heads=2, head_dim=128, page_size=16, n_pages=4, page_stride=4096,
             token_stride=256, head_stride=128, k_scale=1.0, v_scale=1.0)
    a.update(kw)
    return _native.KvCache(**a)


def _scales(**kw):
    a = dict(d_k=P, d_v=2 * P, block=8, page_stride=4, block_stride=2, head_stride=1)
    a.update(kw)
    return _native.KvScales(**a)


def _read(**kw):
    a = dict(d_tables=P, table_stride=4, max_pages=4, requests=2, d_starts=P, d_first=None, tokens=5, d_k_out=P, d_v_out=2 * P,
             k_stride=256, v_stride=256, out_dtype=DType.BF16)
    a.update(kw)
    return _native.KvReadArgs(**a)


CACHES = [
    (dict(dtype=5), {}, NO, "cache"), (dict(d_k=None), {}, BAD, "d_k"), (dict(head_dim=0), {}, BAD, "head_dim"),
    (dict(token_stride=8), {}, BAD, "token_stride"), (dict(k_scale=0.5), {}, BAD, "k_scale"), (dict(v_scale=2.0), {}, BAD, "v_scale"),
    ({}, dict(d_k=None), BAD, "scales d_k"), ({}, dict(d_v=P + 2), BAD, "aligned"), ({}, dict(block=0), BAD, "block"),
    ({}, dict(block=64), BAD, "block"), ({}, dict(block=12), BAD, "block"), ({}, dict(block=32), BAD, "multiple of the block"),
    (dict(page_size=24), dict(block=16), BAD, "multiple of the block"),
    ({}, dict(page_stride=3), BAD, "share an element"), ({}, dict(block_stride=1), BAD, "share an element"),
    ({}, dict(head_stride=0), BAD, "share an element"), ({}, dict(page_stride=-4), BAD, "share an element"),
    ({}, dict(page_stride=1 << 41), BAD, "share an element"), (dict(kv_heads=3), {}, BAD, "share an element")]


@pytest.mark.parametrize("cache,scales,status,word", CACHES)
def test_cache_refusals(cache, scales, status, word):
    _refused(_native.lib().openmini_kv_read(_cache(**cache), _scales(**scales), _read(), None), status, word)


@pytest.mark.parametrize("kw,word", [
    (dict(requests=0), "requests"), (dict(requests=(1 << 20) + 1), "requests"), (dict(tokens=-1), "tokens"), (dict(max_pages=0), "max_pages"),
    (dict(table_stride=3), "table_stride"), (dict(d_tables=None), "d_tables"), (dict(d_starts=None), "d_starts"),
    (dict(d_first=P + 2), "aligned"), (dict(d_k_out=None, d_v_out=None), "both null"), (dict(d_k_out=P + 8), "aligned"),
    (dict(k_stride=248), "k_stride"), (dict(v_stride=260), "v_stride")])
def test_read_refusals(kw, word):
    _refused(_native.lib().openmini_kv_read(_cache(), _scales(), _read(**kw), None), BAD, word)


def test_null_and_mixed_arguments():
    L = _native.lib()
    _refused(L.openmini_kv_read(None, None, None, None), BAD, "null arguments")
    _refused(L.openmini_kv_read(None, None, _read(), None), BAD, "null cache")
    _refused(L.openmini_kv_read(_cache(), None, _read(), None), BAD, "null scales")
    _refused(L.openmini_kv_read(_cache(dtype=DType.BF16), _scales(), _read(), None), BAD, "scales for a cache")
    _refused(L.openmini_kv_read(_cache(), _scales(), _read(out_dtype=DType.I8), None), NO, "k_out")
    _refused(L.openmini_attn_prompt(None, None, None, None), BAD, "null arguments")
    _refused(L.openmini_attn_prompt(None, None, _prompt(), None), BAD, "null cache")
    _refused(L.openmini_attn_prompt(_cache(), None, _prompt(), None), BAD, "null scales")
    _refused(L.openmini_attn_prompt(_cache(dtype=DType.F8_E4M3), _scales(), _prompt(), None), BAD, "scales for a cache")
    _refused(L.openmini_rope_append_i8(None, None, None, None, None), BAD, "null arguments")
    _refused(L.openmini_rope_append_i8(None, _cache(), _scales(), _native.RopeAppendArgs(), None), BAD, "null rope")
    _refused(L.openmini_attn_decode_i8(None, None, None, None), BAD, "null arguments")
    _refused(L.openmini_attn_decode_i8(_cache(), None, _native.AttnArgs(), None), BAD, "null scales")
    _refused(L.openmini_attn_decode_i8(_cache(dtype=DType.BF16), _scales(), _native.AttnArgs(), None), NO, "cache")
    # the calls without scales take no 8-bit integers
    _refused(L.openmini_attn_decode(_cache(), _native.AttnArgs(), None), NO, "cache")


def _prompt(**kw):
    a = dict(d_q=P, q_stride=512, d_out=2 * P, out_stride=512, d_lse=None, q_dtype=DType.BF16, out_dtype=DType.BF16, q_heads=4,
             scale=0.1, window=0, rows=1, d_lens=3 * P, d_starts=5 * P, d_tables=4 * P, table_stride=4, max_pages=4, requests=1,
             d_work=8 * P, work_bytes=1 << 40)
    a.update(kw)
    return _native.PromptArgs(**a)


@pytest.mark.parametrize("cache,args,status,word", [
    (dict(head_dim=80), {}, NO, "head_dim"), (dict(page_size=12, dtype=DType.BF16), {}, NO, "page_size"),
    (dict(dtype=DType.F16), {}, NO, "cache of type 1"), ({}, dict(q_dtype=DType.F32), NO, "q"), ({}, dict(q_dtype=DType.I8), NO, "q"),
    ({}, dict(out_dtype=DType.F16), NO, "out"), ({}, dict(q_heads=3), BAD, "q_heads"), ({}, dict(q_heads=0), BAD, "q_heads"),
    ({}, dict(q_heads=2048), BAD, "q_heads"), ({}, dict(rows=-1), BAD, "rows"), ({}, dict(rows=(1 << 20) + 1), BAD, "rows"),
    ({}, dict(requests=0), BAD, "requests"), ({}, dict(requests=(1 << 20) + 1), BAD, "requests"), ({}, dict(d_q=None), BAD, "d_q"),
    ({}, dict(d_q=P + 2), BAD, "aligned"), ({}, dict(d_out=P), BAD, "d_out is d_q"), ({}, dict(d_lens=None), BAD, "d_lens"),
    ({}, dict(d_starts=None), BAD, "d_starts"), ({}, dict(d_tables=None), BAD, "d_tables"), ({}, dict(q_stride=504), BAD, "q_stride"),
    ({}, dict(out_stride=516), BAD, "out_stride"), ({}, dict(scale=float("nan")), BAD, "scale"), ({}, dict(window=-1), BAD, "window"),
    ({}, dict(max_pages=0), BAD, "max_pages"), ({}, dict(table_stride=3), BAD, "table_stride"), ({}, dict(d_work=None), BAD, "d_work"),
    ({}, dict(d_work=8 * P + 128), BAD, "aligned"), ({}, dict(work_bytes=1000), BAD, "workspace"), ({}, dict(d_lse=P + 1), BAD, "d_lse")])
def test_prompt_refusals(cache, args, status, word):
    c = _cache(**cache)
    s = _scales() if c.dtype == DType.I8 else None
    _refused(_native.lib().openmini_attn_prompt(c, s, _prompt(**args), None), status, word)


def test_calls_past_a_launch():
    """Workgroups of more than 2^32 threads together."""
    c = _cache(dtype=DType.BF16, kv_heads=64, head_dim=128)
    args = _prompt(q_heads=64, q_stride=8192, out_stride=8192, rows=1, requests=1 << 20)
    _refused(_native.lib().openmini_attn_prompt(c, None, args, None), BAD, "too many")
    _refused(_native.lib().openmini_kv_read(_cache(), _scales(), _read(tokens=(1 << 26) + 1), None), BAD, "tokens")


def test_prompt_workspace_bytes():
    L = _native.lib()
    assert L.openmini_attn_prompt_workspace_bytes(64, 8, 128) > 0
    for bad in ((0, 0, 128), (4, 0, 128), (4, 3, 128), (4, 8, 128), (4, 4, 100), (2048, 8, 128), (-4, -2, 128)):
        assert L.openmini_attn_prompt_workspace_bytes(*bad) == 0, bad


@pytest.mark.parametrize("kw,word", [
    (dict(d_k_out=16 * P, d_v_out=16 * P), "d_k_out is d_v_out"), (dict(d_k_out=P, d_v_out=None), "output is the cache"),
    (dict(d_k_out=None, d_v_out=2 * P), "output is the cache"), (dict(d_k_out=16 * P, d_v_out=P), "output is the cache")])
def test_read_over_itself(kw, word):
    _refused(_native.lib().openmini_kv_read(_cache(), _scales(), _read(**kw), None), BAD, word)


def test_prompt_lse_over_others():
    for args in (dict(d_lse=2 * P), dict(d_lse=P)):
        _refused(_native.lib().openmini_attn_prompt(_cache(), _scales(), _prompt(**args), None), BAD, "d_lse is")


def test_strides_whose_sum_passes_63_bits():
    """Scales that share an element behind a stride too far for 64 bits: refused, not wrapped around."""
    c = _cache(n_pages=(1 << 27) - 1)
    far = _scales(page_stride=1 << 37, block_stride=1 << 40, head_stride=1)
    _refused(_native.lib().openmini_kv_read(c, far, _read(), None), BAD, "share an element")


class Buf:
    ptr, nbytes = ctypes.c_void_p(P), 1 << 20


class Short:
    ptr, nbytes = ctypes.c_void_p(P), 60


def test_mirror_refusals():
    with pytest.raises(InvalidInput, match="needs d_k_scales"):
        KVCache(Buf, Buf, DType.I8, 4, 16, 2, 128, block=8)
    with pytest.raises(InvalidInput, match="whole blocks"):
        KVCache(Buf, Buf, DType.I8, 4, 16, 2, 128, d_k_scales=Buf, d_v_scales=Buf)
    with pytest.raises(InvalidInput, match="whole blocks"):
        KVCache(Buf, Buf, DType.I8, 4, 24, 2, 128, block=16, d_k_scales=Buf, d_v_scales=Buf)
    with pytest.raises(InvalidInput, match="d_v_scales"):
        KVCache(Buf, Buf, DType.I8, 4, 16, 2, 128, block=8, d_k_scales=Buf, d_v_scales=Short)
    with pytest.raises(InvalidInput, match="blocks with scales"):
        KVCache(Buf, Buf, DType.BF16, 4, 16, 2, 128, block=8)
    assert DType.of("i8").nbytes == 1
    for layout, want in (("token", (4, 2, 1)), ("head", (4, 1, 2))):
        c = KVCache(Buf, Buf, DType.I8, 4, 16, 2, 128, layout=layout, block=8, d_k_scales=Buf, d_v_scales=Buf)
        assert (c.scales.page_stride, c.scales.block_stride, c.scales.head_stride) == want
    for args in ((Short, 4, Buf, 4, 2, Buf, Buf), (Buf, 4, Buf, 15, 2, Short, Buf), (Buf, 4, Short, 15, 2, Buf, Buf),
                 (Buf, 4, Buf, 4, 2, Buf, Short)):
        with pytest.raises(InvalidInput, match="are needed"):
            c.read(args[0], args[1], args[2], args[3], args[4], args[5], args[6], DType.F32, d_first=None)
    p = PromptAttention.__new__(PromptAttention)
    p.q_heads, p.kv_heads, p.head_dim, p.window, p.scale = 4, 2, 128, 0, 0.1
    p.q_dtype, p.out_dtype, p.work, p._call = DType.BF16, DType.BF16, Buf, None
    good = dict(cache=c, d_q=Buf, d_out=Buf, d_tables=Buf, max_pages=4, d_starts=Buf, d_lens=Buf, rows=20, requests=15)
    for name in ("d_q", "d_out", "d_tables", "d_starts", "d_lens"):
        with pytest.raises(InvalidInput, match=name):
            p.run(**{**good, name: Short})
    with pytest.raises(InvalidInput, match="d_lse"):
        p.run(**good, d_lse=Short)
    other = KVCache(Buf, Buf, DType.I8, 4, 16, 1, 128, block=8, d_k_scales=Buf, d_v_scales=Buf)
    with pytest.raises(InvalidInput, match="expected 2"):
        p.run(**{**good, "cache": other})
