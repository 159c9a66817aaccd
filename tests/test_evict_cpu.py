"""Argument checks of the eviction, accumulation and norm-and-rotate C entries, which need no GPU."""
import ctypes

import pytest
import torch

import snapmind_b200._lib as lib

X = ctypes.c_void_p(256)


def evict(pool_dtype=1, scales=None, n=2, budget=8, recent=0, sinks=0, layers=1, heads=2, d=64, bs=16, nb=4, width=4, k=None,
          seqs=None, into=None):
    return lib.load().snapmind_kv_evict_by_mass(
        k, k, scales, pool_dtype, 0, 0, k, 0, k, 0, width, k, seqs, into, n, budget, recent, sinks, 0, k, k, k, layers, heads,
        d, bs, nb, None, None)


@pytest.mark.parametrize("kw,word", [
    (dict(pool_dtype=9), "dtype"),
    (dict(pool_dtype=lib.DTYPE_E4M3), "scales"),
    (dict(scales=X), "scales"),
    (dict(n=-1), "sizes"),
    (dict(layers=0), "sizes"),
    (dict(heads=0), "sizes"),
    (dict(bs=0), "sizes"),
    (dict(budget=0), "budget"),
    (dict(recent=5, sinks=4), "budget"),
    (dict(recent=2**31 - 1, sinks=2**31 - 1), "budget"),
    (dict(recent=-1), "budget"),
    (dict(width=1 << 28), "too long"),
    (dict(n=1 << 30, layers=64), "too many"),
    (dict(), "null"),
    (dict(k=X, into=X), "named"),
])
def test_evict_refusals(kw, word):
    assert evict(**kw) == lib.ERR_BAD_ARGUMENT
    assert word in lib.last_error()


def test_evict_of_nothing():
    assert evict(n=0) == lib.OK


def clear(batch=1, n=1, layers=1, counts=None):
    return lib.load().snapmind_kv_clear_mass(None, 0, None, 0, 4, None, counts, n, batch, layers, 2, 16, 4, None, None)


def test_clear_refusals():
    for kw in (dict(batch=-1), dict(n=-1), dict(layers=0), dict()):
        assert clear(**kw) == lib.ERR_BAD_ARGUMENT
    assert clear(batch=0) == lib.OK and clear(n=0) == lib.OK


def test_mass_workspace():
    ws = lib.load().snapmind_paged_gqa_chunk_mass_workspace_bytes
    plain = lib.load().snapmind_paged_gqa_chunk_workspace_bytes(128)
    assert ws(128, 10, 32, 8, 16, 100, 0) > plain
    # a decode on the kernel that keeps its scores: one for every slot and query head
    assert ws(128, 10, 32, 8, 16, 100, 1) == ws(128, 10, 32, 8, 16, 100, 0) + 100 * 16 * 32 * 4
    assert ws(64, 10, 32, 8, 16, 100, 1) == ws(64, 10, 32, 8, 16, 100, 0)
    for bad in ((0, 1, 1, 1, 16, 4, 0), (257, 1, 1, 1, 16, 4, 0), (128, -1, 1, 1, 16, 4, 0), (128, 1, 0, 1, 16, 4, 0), (128, 1, 1, 0, 16, 4, 0)):
        assert ws(*bad) == 0


def rope(dtype=1, pool_dtype=1, scales=None, batch=2, total=2, hq=2, hkv=2, d=64, rot=64, n_pos=8, eps=0.0, cu=None, bs=16, x=None):
    return lib.load().snapmind_norm_rope_append(
        x, 0, 0, x, 0, 0, hq, x, 0, 0, x, 0, 0, dtype, None, 0, None, 0, eps, x, x, rot, n_pos, None, x, x, scales, pool_dtype,
        x, 0, 4, x, cu, batch, total, hkv, d, bs, 4, None, None)


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=7), "dtype"),
    (dict(pool_dtype=7), "dtype"),
    (dict(pool_dtype=lib.DTYPE_E4M3), "scales"),
    (dict(scales=X), "scales"),
    (dict(batch=3), "one token"),
    (dict(hkv=0), "sizes"),
    (dict(bs=0), "sizes"),
    (dict(n_pos=0), "sizes"),
    (dict(batch=1 << 29, total=1 << 29), "sizes"),
    (dict(rot=66), "rotated"),
    (dict(rot=31), "rotated"),
    (dict(rot=-2), "rotated"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(), "null"),
    (dict(x=X), "null"),  # no positions
])
def test_append_rope_refusals(kw, word):
    assert rope(**kw) == lib.ERR_BAD_ARGUMENT
    assert word in lib.last_error()


def test_append_rope_of_nothing():
    assert rope(batch=0, total=0) == lib.OK


def chunk_mass(total=8, width=4, mass=256, dtype=0, x=X):
    return lib.load().snapmind_paged_gqa_chunk_mass(x, 512, 64, dtype, x, x, None, dtype, x, width, width, x, x, x, 512, 64, 1.0, 1,
                                                    total, 8, 1, 64, 16, 4, 0, 0, 0, ctypes.c_void_p(mass), x, 1 << 60, None, None)


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up pointers")
@pytest.mark.parametrize("kw,word", [
    (dict(total=1 << 22, width=1 << 22), "too many"),
    (dict(total=1 << 30, width=1 << 16), "too many"),
    (dict(mass=260), "16-byte"),
])
def test_accumulate_refusals(kw, word):
    """All before the attention of the call is launched."""
    assert chunk_mass(**kw) == lib.ERR_BAD_ARGUMENT
    assert word in lib.last_error()
