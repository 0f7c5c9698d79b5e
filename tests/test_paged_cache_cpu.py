"""The paged cache's C entries refuse what they cannot run, before any launch."""
import ctypes

import pytest

from megalodon_amd import _lib

i64, p8 = ctypes.c_int64, ctypes.POINTER(ctypes.c_uint8)


class Cache(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_exponents", ctypes.c_void_p), ("v_exponents", ctypes.c_void_p),
                ("k_stride", i64 * 3), ("v_stride", i64 * 3), ("ke_stride", i64 * 3), ("ve_stride", i64 * 3),
                ("pages", i64), ("page_size", i64), ("heads", i64), ("k_width", i64), ("v_width", i64),
                ("table", ctypes.c_void_p), ("table_stride", i64), ("table_width", i64), ("batch", i64)]


def cache(**changes):
    c = Cache(k=1 << 20, v=1 << 21, k_stride=(i64 * 3)(4096, 256, 128), v_stride=(i64 * 3)(4096, 256, 128), pages=10, page_size=16, heads=2,
              k_width=128, v_width=128, table=1 << 22, table_stride=4, table_width=4, batch=3)
    for name, value in changes.items():
        setattr(c, name, (i64 * 3)(*value) if isinstance(value, tuple) else value)
    return c


def code(fn, *args):
    fn = getattr(_lib.load(), fn)
    fn.restype = ctypes.c_int
    return fn(*args)


def attend(c, dtype=1, q=1 << 16, q_row=256, q_head=128, lengths=1 << 8, cu=1 << 9, rows=5, q_heads=2, scale=1.0, chunk=0, out=1 << 17, workspace=None):
    return code("mega_paged_attention_fwd", ctypes.byref(c) if c is not None else None, ctypes.c_int(dtype), ctypes.c_void_p(q), i64(q_row), i64(q_head),
                ctypes.c_void_p(lengths), ctypes.c_void_p(cu), i64(rows), i64(q_heads), ctypes.c_double(scale), i64(chunk), ctypes.c_void_p(out),
                ctypes.c_int(1), ctypes.c_void_p(workspace), None)


def write(c, dtype=1, k=1 << 16, k_row=256, k_head=128, v=1 << 17, v_row=256, v_head=128, lengths=1 << 8, cu=1 << 9, rows=5):
    return code("mega_paged_cache_write", ctypes.byref(c), ctypes.c_int(dtype), ctypes.c_void_p(k), i64(k_row), i64(k_head), ctypes.c_void_p(v), i64(v_row),
                i64(v_head), ctypes.c_void_p(lengths), ctypes.c_void_p(cu), i64(rows), None)


def read(c, dtype=1, begins=1 << 8, cu=1 << 9, rows=5, k=1 << 16, v=1 << 17):
    return code("mega_paged_cache_read", ctypes.byref(c), ctypes.c_int(dtype), ctypes.c_void_p(begins), ctypes.c_void_p(cu), i64(rows), ctypes.c_void_p(k),
                ctypes.c_void_p(v), ctypes.c_int(1), None)


BAD_CACHES = [dict(k=None), dict(v=None), dict(k=(1 << 20) + 8), dict(pages=0), dict(pages=1 << 31), dict(page_size=8), dict(page_size=24),
              dict(page_size=1 << 17), dict(heads=0), dict(k_width=0), dict(k_width=24), dict(v_width=4112), dict(table=None), dict(table_width=1 << 28),
              dict(batch=-1), dict(k_stride=(4096, 256, 120)), dict(v_stride=(4096, -256, 128)), dict(v_stride=(4096, 1 << 28, 128)),
              dict(k_exponents=1 << 10), dict(v_exponents=1 << 10), dict(k_exponents=1 << 10, v_exponents=1 << 11, ke_stride=(32, 2, -1))]


@pytest.mark.parametrize("changes", BAD_CACHES, ids=str)
def test_caches_that_are_refused(changes):
    c = cache(**changes)
    assert attend(c) == 1 and write(c) == 1 and read(c) == 1
    assert b"mega_paged_cache_read" in _lib.load().mega_last_error()


@pytest.mark.parametrize("bad", [dict(dtype=0), dict(dtype=3), dict(q=None), dict(q=(1 << 16) + 2), dict(q_row=100), dict(lengths=None), dict(cu=None),
                                 dict(rows=-1), dict(rows=1 << 31), dict(q_heads=3), dict(q_heads=0), dict(chunk=-1), dict(out=None), dict(out=(1 << 17) + 8)], ids=str)
def test_attention_calls_that_are_refused(bad):
    assert attend(cache(), **bad) == 1
    assert b"mega_paged_attention_fwd" in _lib.load().mega_last_error()


def test_attention_wants_its_workspace():
    c, lib = cache(table_width=1000), _lib.load()
    lib.mega_paged_attention_workspace_bytes.restype = i64
    size = lib.mega_paged_attention_workspace_bytes(ctypes.byref(c), i64(5), i64(2), i64(0))
    assert size > 0
    assert attend(c) == 1 and b"workspace" in lib.mega_last_error()
    for rows, heads, chunk in ((0, 2, 0), (-1, 2, 0), (5, 3, 0), (5, 2, -1)):
        assert lib.mega_paged_attention_workspace_bytes(ctypes.byref(c), i64(rows), i64(heads), i64(chunk)) == 0
    assert lib.mega_paged_attention_workspace_bytes(None, i64(5), i64(2), i64(0)) == 0
    wide = cache(k_width=528, k_stride=(32 * 528, 1056, 528))
    assert attend(wide, q_head=528, q_row=1056) == 1 and b"512" in lib.mega_last_error()


@pytest.mark.parametrize("bad", [dict(dtype=0), dict(k=None), dict(v=None), dict(k=(1 << 16) + 2), dict(k_row=100), dict(v_head=4), dict(lengths=None),
                                 dict(cu=None), dict(rows=-1)], ids=str)
def test_writes_that_are_refused(bad):
    assert write(cache(), **bad) == 1


@pytest.mark.parametrize("bad", [dict(dtype=0), dict(k=None), dict(v=None), dict(v=(1 << 17) + 2), dict(begins=None), dict(cu=None), dict(rows=-1)], ids=str)
def test_reads_that_are_refused(bad):
    assert read(cache(), **bad) == 1


def test_calls_of_nothing_launch_nothing():
    assert attend(cache(), rows=0) == 0 and write(cache(), rows=0) == 0 and read(cache(), rows=0) == 0 and write(cache(batch=0)) == 0


def test_a_table_row_holds_up_to_two_to_the_30_positions():
    c = cache(table_width=(1 << 26) + 1)
    assert attend(c) == 1 and b"2^30" in _lib.load().mega_last_error()
    assert write(c) == 1 and read(c) == 1


def test_questions_leave_the_last_error():
    lib = _lib.load()
    assert attend(cache(), dtype=7) == 1
    before = lib.mega_last_error()
    lib.mega_paged_attention_workspace_bytes(ctypes.byref(cache()), i64(5), i64(3), i64(0))
    assert lib.mega_last_error() == before
