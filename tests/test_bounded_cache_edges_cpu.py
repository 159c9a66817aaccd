"""Argument checks of the bounded cache's C entries, which need no GPU."""
import ctypes

import snapmind_b200._lib as lib

X = ctypes.c_void_p(256)


def reserve(tables=X, counts=None, n=1, batch=1, bs=16, width=4):
    return lib.load().snapmind_kv_reserve_status(tables, width, width, tables, counts, n, batch, bs, tables, tables, 4, None, None, None)


def test_reserve_status_refusals():
    for kw in (dict(batch=-1), dict(n=-1), dict(bs=0), dict(width=-1)):
        assert reserve(**kw) == lib.ERR_BAD_ARGUMENT and "sizes" in lib.last_error()
    assert reserve(tables=None) == lib.ERR_BAD_ARGUMENT and "null" in lib.last_error()
    assert reserve(batch=0) == reserve(tables=None, batch=0) == lib.OK
