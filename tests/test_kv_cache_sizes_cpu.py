"""Sizes at the C entries of the key/value cache, on the host: what they refuse, and the workspaces they ask for."""
import ctypes
import struct
import subprocess
import sys

from conftest import PKG_PARENT

BIG = 2 ** 64 - 1


def _lib():
    from h3vae_b200 import _lib, build_lib
    build_lib.build()
    return _lib, _lib.load()


def test_workspace_sizes_of_any_sizes_come_back():
    """Sizes far past what a call takes: a number comes back (a child process, since a division by zero would end it)."""
    _lib()
    code = f"""
import sys
sys.path.insert(0, {str(PKG_PARENT)!r})
from h3vae_b200 import _lib
lib = _lib.load()
small = (1, 2, 2, 60, 64, 40, 16, 0)
for i in range(8):
    for big in (1 << 62, 1 << 57, (1 << 63) - 1, 1 << 33, 0, -1, -(1 << 63)):
        for other in range(8):
            for second in (small[other], 1 << 57, 1 << 32):
                sizes = list(small)
                sizes[other], sizes[i] = second, big
                assert lib.h3b_attention_kv_i8_workspace_size(*sizes) >= 16
                assert lib.h3b_kv_select_i8_workspace_size(*sizes[:1], *sizes[2:4], sizes[5]) >= 16
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert done.returncode == 0, (done.returncode, done.stderr[-500:])


def test_workspace_sizes_do_not_wrap():
    """Products past 64 bits: no workspace is large enough, and never a small number."""
    _, lib = _lib()
    assert lib.h3b_kv_select_i8_workspace_size(1 << 16, 1 << 16, 1 << 16, 1 << 16) == BIG
    assert lib.h3b_kv_select_i8_workspace_size(1 << 14, 1 << 14, 1 << 20, 1 << 14) == BIG
    assert lib.h3b_kv_select_i8_workspace_size(1 << 15, 1 << 14, 1 << 10, 1 << 12) == 1 << 53
    assert lib.h3b_attention_kv_i8_workspace_size(65535, 65535, 65535, 16384, 128, 1 << 26, 16, 1 << 20) == BIG
    assert lib.h3b_attention_kv_i8_workspace_size(65535, 65535, 65535, 1, 128, 1 << 26, 16, 0) > 1 << 47


def test_workspace_sizes_follow_the_plan():
    """16 where the blocks of a cluster join (the call takes no workspace); room for every part's row, maximum and sum
    where a second kernel joins: at most as many runs as the device holds blocks, one a sequence at least."""
    _, lib = _lib()

    def size(batch=1, q_heads=16, kv_heads=16, tokens=1, dim=64, width=100, page=64, n=0):
        return lib.h3b_attention_kv_i8_workspace_size(batch, q_heads, kv_heads, tokens, dim, width, page, n)

    assert size(width=29) == size(width=8) == 16 and size(width=1000, n=32) == 16
    for dim in (64, 128):
        one = size(width=2048, dim=dim)                  # 131072 keys of 16 heads
        part = 16 * 16 * (dim + 4) * 4
        assert one > 16 + 2 * part and (one - 32) % part == 0
        assert size(batch=16, width=2048, dim=dim) > 16 * part
        assert size(tokens=128, width=512, dim=dim) > 16 + 2 * 16 * 128 * (dim + 4) * 4      # row tiles, parts of keys


def test_sizes_past_the_limits_are_refused():
    """Pointers here are never followed: every call is refused on the host."""
    mod, lib = _lib()
    st = struct.pack("3q", 0, 0, 64)

    def cache(**kw):
        fields = dict(k=64, v=64, k_scale=64, v_scale=64, k_sum=64, num_pages=4, kv_heads=2, page_size=16, head_dim=64)
        return ctypes.byref(mod.KvCacheStruct(**{**fields, **kw}))

    def store(c, width, tokens=1):
        yield lib.h3b_kv_write_i8(c, 64, 1, width, 64, None, 64, st, 64, st, tokens, 0, None)
        yield lib.h3b_kv_read_i8(c, 64, 1, width, None, 64, 64, 64, tokens, 0, None)

    def query(c, width, tokens=1, heads=4):
        yield lib.h3b_attention_kv_i8(64, st, c, 64, 1, width, 64, None, heads, tokens, 1.0, 1, 0, None, 0, 0, 64, st, None,
                                      64, BIG, None)
        yield lib.h3b_kv_select_i8(64, st, c, 64, 1, width, 64, None, heads, tokens, 4, 0, 64, 64, BIG, None)

    for width in (1 << 60, 1 << 59, (1 << 62) + 1, (1 << 26) + 1):
        assert {*store(cache(), width), *query(cache(), width)} == {mod.H3B_EUNSUPPORTED}, width
    refused = {mod.H3B_EINVAL, mod.H3B_EUNSUPPORTED}
    for tokens in (1 << 62, (1 << 63) - 1, 1 << 50):
        assert {*store(cache(), 2, tokens), *query(cache(), 2, tokens)} <= refused, tokens
    for heads in (1 << 62, 1 << 32, 65536):
        assert set(query(cache(), 2, heads=heads)) <= refused, heads
