"""Argument checks of the bounded cache's C entries, which need no GPU."""
import ctypes

import pytest
import torch

import snapmind_b200._lib as lib

X = ctypes.c_void_p(256)


def reserve(tables=X, counts=None, n=1, batch=1, bs=16, width=4):
    return lib.load().snapmind_kv_reserve_status(tables, width, width, tables, counts, n, batch, bs, tables, tables, 4, None, None, None)


def test_reserve_status_refusals():
    for kw in (dict(batch=-1), dict(n=-1), dict(bs=0), dict(width=-1)):
        assert reserve(**kw) == lib.ERR_BAD_ARGUMENT and "sizes" in lib.last_error()
    assert reserve(tables=None) == lib.ERR_BAD_ARGUMENT and "null" in lib.last_error()
    assert reserve(batch=0) == reserve(tables=None, batch=0) == lib.OK


def evict(mass=256, layer=1024, bs=16):
    return lib.load().snapmind_kv_evict_by_mass(
        X, X, None, 1, 4096, 0, ctypes.c_void_p(mass), layer, X, 4, 4, X, None, None, 1, 8, 0, 0, 0, X, X, X, 2, 2, 64, bs, 4, None, None)


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up pointers")
@pytest.mark.parametrize("kw", [dict(mass=260), dict(mass=264), dict(layer=1022), dict(layer=1025, bs=4)])
def test_evict_refuses_weights_off_their_boundary(kw):
    """Weights of blocks of a multiple of 4 tokens, which are read four at a time."""
    assert evict(**kw) == lib.ERR_BAD_ARGUMENT and "16-byte" in lib.last_error()
