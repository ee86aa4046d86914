"""Refusals of the scoring and paging operators, on the host: the library validates before any launch (the pointers here
are dummies), the Python entry points before any library call."""
import ctypes

import pytest
import torch

from palu_b200 import _lib, build, paging, scoring

I = ctypes.c_int32


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def arr(*x):
    return (I * len(x))(*x)


@pytest.mark.parametrize("change,needle", [
    (dict(rows=-1), "rows"), (dict(vocab=0), "vocab"), (dict(dtype=7), "dtype"), (dict(top=33), "top"), (dict(top=-1), "top"),
    (dict(vocab=10, top=11), "top"), (dict(ld=99), "cannot hold"), (dict(logits=None), "must be set"),
    (dict(top_id=None), "must be set"), (dict(logits=17), "aligned"),
])
def test_logprob_refusals(lib, change, needle):
    a = dict(logits=16, ld=100, dtype=_lib.PALU_BF16, rows=4, vocab=100, tokens=16, t64=1, top=5, lp=16, ent=16, tv=16, top_id=16)
    a.update(change)
    st = lib.palu_token_logprobs(*a.values(), None)
    assert st == _lib.PALU_ERR_INVALID and needle in lib.palu_last_error().decode()


def test_python_refusals():
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        scoring.token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.long))
    cache = torch.zeros(4, 1, 16, 8)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        paging.copy_pages([cache], [0], [1])
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        paging.PagePool([cache], rows=1, blocks_per_row=1)
    with pytest.raises(RuntimeError, match="at least one cache"):
        paging.copy_pages([], [0], [1])
    with pytest.raises(RuntimeError, match="32 bits"):
        paging._ints([1 << 33], "rows")


def pool(**kw):
    a = dict(table=16, refs=16, mapped=16, status=16, rows=4, blocks_per_row=3, n_blocks=9, block_size=16)
    a.update(kw)
    return ctypes.byref(_lib.PagePoolInfo(**a))


CACHE = (_lib.PageCache * 1)(_lib.PageCache(16, 64, 64))


@pytest.mark.parametrize("p,needle", [(dict(table=None), "must be set"), (dict(status=None), "must be set"), (dict(rows=0), "positive"), (dict(rows=1 << 16, blocks_per_row=1 << 15), "entries"),
                                      (dict(block_size=-1), "positive")])
def test_pool_refusals(lib, p, needle):
    for st in (lib.palu_reserve_pages(pool(**p), arr(0), arr(1), 1, None), lib.palu_free_pages(pool(**p), arr(0), 1, None),
               lib.palu_fork_pages(pool(**p), CACHE, 1, arr(0), arr(1), arr(1), 1, 16, 1 << 20, None),
               lib.palu_compact_pages(pool(**p), CACHE, 1, 16, 1 << 20, None)):
        assert st == _lib.PALU_ERR_INVALID and needle in lib.palu_last_error().decode()


@pytest.mark.parametrize("rows,lens,needle", [((4,), (1,), "outside"), ((-1,), (1,), "outside"), ((0, 0), (1, 2), "twice"),
                                              ((0,), (49,), "cannot hold"), ((0,), (-1,), "cannot hold")])
def test_row_refusals(lib, rows, lens, needle):
    st = lib.palu_reserve_pages(pool(), arr(*rows), arr(*lens), len(rows), None)
    assert st == _lib.PALU_ERR_INVALID and needle in lib.palu_last_error().decode()
    st = lib.palu_fork_pages(pool(), CACHE, 1, arr(*[3] * len(rows)), arr(*rows), arr(*lens), len(rows), 16, 1 << 20, None)
    assert st == _lib.PALU_ERR_INVALID and needle in lib.palu_last_error().decode()


def test_fork_refusals(lib):
    st = lib.palu_fork_pages(pool(), CACHE, 1, arr(0, 1), arr(1, 2), arr(5, 5), 2, 16, 1 << 20, None)
    assert st == _lib.PALU_ERR_INVALID and "parent and a child" in lib.palu_last_error().decode()
    st = lib.palu_fork_pages(pool(), CACHE, 1, arr(9), arr(1), arr(5), 1, 16, 1 << 20, None)
    assert st == _lib.PALU_ERR_INVALID and "parents" in lib.palu_last_error().decode()
    need = lib.palu_page_workspace_bytes(9)
    st = lib.palu_fork_pages(pool(), CACHE, 1, arr(0), arr(1), arr(5), 1, 16, need - 1, None)
    assert st == _lib.PALU_ERR_WORKSPACE
    st = lib.palu_compact_pages(pool(), CACHE, 1, None, need, None)
    assert st == _lib.PALU_ERR_WORKSPACE


@pytest.mark.parametrize("src,dst,needle", [((0,), (9,), "outside"), ((-1,), (0,), "outside"), ((0, 1), (2, 2), "twice"),
                                            ((0, 1), (1, 2), "copied from and copied to")])
def test_copy_refusals(lib, src, dst, needle):
    st = lib.palu_copy_pages(CACHE, 1, 9, arr(*src), arr(*dst), len(src), None)
    assert st == _lib.PALU_ERR_INVALID and needle in lib.palu_last_error().decode()


def test_cache_refusals(lib):
    for bad in (_lib.PageCache(None, 64, 64), _lib.PageCache(16, 32, 64), _lib.PageCache(16, 64, 0)):
        st = lib.palu_copy_pages((_lib.PageCache * 1)(bad), 1, 9, arr(0), arr(1), 1, None)
        assert st == _lib.PALU_ERR_INVALID and "cache 0" in lib.palu_last_error().decode()
