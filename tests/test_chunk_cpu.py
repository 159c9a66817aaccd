"""Argument checks of the chunk operators' C entries and of their Python wrappers that need no GPU."""
import ctypes

import pytest
import torch

import snapmind_b200._lib as lib


def chunk(dtype=1, pool_dtype=1, scales=None, batch=1, total=1, hq=8, hkv=8, d=128, bs=16, window=0, sinks=0, cu=None,
          ws_bytes=0):
    return lib.load().snapmind_paged_gqa_chunk(
        None, 0, 0, dtype, None, None, scales, pool_dtype, None, 0, 0, None, cu, None, 0, 0, 1.0, batch, total, hq,
        hkv, d, bs, 4, window, sinks, 0, None, ws_bytes, None, None)


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=7), "dtype"),
    (dict(dtype=1, pool_dtype=2), "e4m3"),
    (dict(pool_dtype=lib.DTYPE_E4M3), "scales"),
    (dict(scales=ctypes.c_void_p(16)), "scales"),
    (dict(hq=7, hkv=2), "multiple"),
    (dict(d=0), "head_dim"),
    (dict(d=257), "head_dim"),
    (dict(bs=0), "sizes"),
    (dict(batch=8193, total=8193), "batch"),
    (dict(batch=-1), "sizes"),
    (dict(window=-1), "negative"),
    (dict(window=4, sinks=-1), "negative"),
    (dict(sinks=4), "window"),
    (dict(batch=2, total=3), "one query"),
    (dict(), "null"),
])
def test_chunk_refusals(kw, word):
    assert chunk(**kw) == lib.ERR_BAD_ARGUMENT
    assert word in lib.last_error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up pointers")
@pytest.mark.parametrize("total,width", [(1 << 30, 1 << 16), (1 << 22, 1 << 22)])
def test_chunk_of_too_much(total, width):
    """The tiles of one kv head are counted in 32 bits: more than that is refused."""
    x = ctypes.c_void_p(256)
    rc = lib.load().snapmind_paged_gqa_chunk(x, 512, 64, 0, x, x, None, 0, x, width, width, x, x, x, 512, 64, 1.0, 1,
                                             total, 8, 1, 64, 16, 4, 0, 0, 0, x, 1 << 60, None, None)
    assert rc == lib.ERR_BAD_ARGUMENT and "too many" in lib.last_error()


def test_chunk_of_nothing():
    assert chunk(batch=0, total=0) == lib.OK
    assert chunk(total=0, cu=ctypes.c_void_p(16)) == lib.OK


def append(pool_dtype=3, scales=ctypes.c_void_p(16), in_dtype=1, batch=2, n_tok=3, total=6, cu=None, layers=1, heads=2):
    return lib.load().snapmind_kv_append_chunk(
        None, None, scales, pool_dtype, 0, 0, None, None, in_dtype, 0, 0, 0, 0, None, 0, 0, None, 0, cu, layers, batch,
        n_tok, total, heads, 64, 16, 4, None, None)


@pytest.mark.parametrize("kw,word", [
    (dict(in_dtype=3), "dtype"),
    (dict(pool_dtype=4), "dtype"),
    (dict(scales=None), "scales"),
    (dict(pool_dtype=1), "scales"),
    (dict(total=5), "n_tokens"),
    (dict(layers=-1), "sizes"),
    (dict(batch=1 << 20, n_tok=1 << 10, total=1 << 30, heads=2), "rows"),
    (dict(), "null"),
])
def test_append_refusals(kw, word):
    assert append(**kw) == lib.ERR_BAD_ARGUMENT
    assert word in lib.last_error()


def test_append_of_nothing():
    assert append(batch=0, n_tok=3, total=0) == lib.OK


def test_gather_and_reserve_refusals():
    l = lib.load()
    args = [None, None, None, 0, 0, None, None, 1, 0, 0, None, 0, 0, None, 1, 1, 1, 64, 16, 4, None, None]
    assert l.snapmind_kv_gather_quant(*args) == lib.ERR_BAD_ARGUMENT and "null" in lib.last_error()
    assert l.snapmind_kv_gather_quant(*args[:7], 3, *args[8:]) == lib.ERR_BAD_ARGUMENT and "dtype" in lib.last_error()
    assert l.snapmind_kv_gather_quant(*args[:15], 9000, *args[16:]) == lib.ERR_BAD_ARGUMENT and "sizes" in lib.last_error()
    assert l.snapmind_kv_reserve_each(None, 0, 0, None, None, 1, 16, None, None, 4, None, None) == lib.ERR_BAD_ARGUMENT
    assert l.snapmind_kv_reserve_each(None, 0, 0, None, None, 0, 16, None, None, 4, None, None) == lib.OK


def test_workspace_bytes():
    l = lib.load()
    assert l.snapmind_paged_gqa_chunk_workspace_bytes(128) % 256 == 0
    assert l.snapmind_paged_gqa_chunk_workspace_bytes(0) == 0
    assert l.snapmind_paged_gqa_chunk_workspace_bytes(257) == 0


def test_offsets_are_checked():
    ok = torch.zeros(3, dtype=torch.int32)
    lib.require_offsets("x", ok, ok)
    for bad in (ok.long(), ok.view(1, 3), ok[:0], torch.zeros(6, dtype=torch.int32)[::2], ok.to("meta")):
        with pytest.raises(ValueError):
            lib.require_offsets("x", bad, ok)
