"""What of the key/value cache needs no GPU: the library's exports and its refusals, which come before any launch."""
import ctypes
import re
import struct

from conftest import ROOT


def _lib():
    from h3vae_b200 import _lib, build_lib
    build_lib.build()
    return _lib, _lib.load()


def test_exports_match_the_header():
    lib_mod, lib = _lib()
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "h3vae_b200_kv.h").read_text(), flags=re.S)
    names = set(re.findall(r"\b(h3b_[a-z0-9_]+)\s*\(", text))
    assert names == set(lib_mod._KV_SIGNATURES) and all(hasattr(lib, n) for n in names)
    assert names <= set(lib_mod.EXPORTED_SYMBOLS)


def _cache(lib_mod, **kw):
    fields = dict(k=64, v=64, k_scale=64, v_scale=64, k_sum=64, num_pages=4, kv_heads=2, page_size=16, head_dim=64)
    fields.update(kw)
    return ctypes.byref(lib_mod.KvCacheStruct(**fields))      # kept alive by the reference


def test_refusals_at_the_c_entries():
    """Pointers here are never followed: every call is refused on the host."""
    lib_mod, lib = _lib()
    st = struct.pack("3q", 0, 0, 64)

    def write(cache, table=64, batch=1, width=2, start=64, k=64, tokens=1, dtype=0):
        return lib.h3b_kv_write_i8(cache, table, batch, width, start, None, k, st, 64, st, tokens, dtype, None)

    def attend(cache, q=64, heads=4, tokens=1, causal=1, window=0, sel=None, n_sel=0, dtype=0, ws=64, ws_bytes=0):
        return lib.h3b_attention_kv_i8(q, st, cache, 64, 1, 2, 64, None, heads, tokens, 1.0, causal, window, sel, n_sel,
                                       dtype, 64, st, None, ws, ws_bytes, None)

    inval, unsup = lib_mod.H3B_EINVAL, lib_mod.H3B_EUNSUPPORTED
    good = _cache(lib_mod)
    assert write(None) == inval and write(_cache(lib_mod, k=None)) == inval and write(good, table=None) == inval
    assert write(_cache(lib_mod, v=72)) == inval and write(_cache(lib_mod, head_dim=80)) == unsup
    assert write(_cache(lib_mod, page_size=48)) == unsup and write(_cache(lib_mod, num_pages=0)) == inval
    assert write(good, batch=0) == inval and write(good, batch=70000) == unsup and write(good, width=1 << 28) == unsup
    assert write(good, start=None) == inval and write(good, k=None) == inval and write(good, dtype=3) == inval
    assert write(good, tokens=-1) == inval and write(good, tokens=0) == 0
    assert "h3b_kv_write_i8" in lib_mod.last_error()
    assert lib.h3b_kv_read_i8(good, 64, 1, 2, None, None, 64, 64, 4, 0, None) == inval
    assert lib.h3b_kv_read_i8(good, 64, 1, 2, None, 64, 64, 65, 4, 0, None) == inval
    assert lib.h3b_kv_read_i8(good, 64, 1, 2, None, 64, 64, 64, 0, 0, None) == 0
    assert attend(good, q=None) == inval and attend(good, heads=3) == inval and attend(good, heads=0) == inval
    assert attend(good, dtype=2) == inval and attend(good, window=-1) == inval and attend(good, causal=0, window=3) == inval
    assert attend(good, sel=64, n_sel=0) == inval and attend(good, causal=0, sel=64, n_sel=1) == inval
    assert attend(good, tokens=0) == 0
    assert lib.h3b_kv_select_i8(64, st, good, 64, 1, 2, 64, None, 4, 1, 0, 0, 64, 64, 64, None) == inval
    assert lib.h3b_kv_select_i8(64, st, good, 64, 1, 2, 64, None, 4, 1, 2, 0, 64, 64, 15, None) == inval


def test_workspace_sizes():
    _, lib = _lib()
    assert lib.h3b_kv_select_i8_workspace_size(2, 3, 4, 5) >= 2 * 3 * 4 * 5 * 4
    assert lib.h3b_attention_kv_i8_workspace_size(1, 16, 16, 1, 64, 100, 64, 0) > 0
