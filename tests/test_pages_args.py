"""Refusals of the page pool's calls that need no GPU."""
import pytest
import torch

from fold_b200 import _lib, kernels
from fold_b200.errors import FoldError

P = 1 << 20


def pool(kw):
    a = dict(refs=P, pages=8, tables=P, stride=4, width=4, lens=P, rows=3)
    a.update({k: kw.pop(k) for k in list(kw) if k in a})
    return list(a.values())


def grow(**kw):
    args = pool(kw)
    a = dict(named=P, qsl=P, m=2, n=4, bs=16, pos=P, slots=P)
    a.update(kw)
    _lib.call("fold_grow_pages", *args, *a.values(), None, None)


def free(**kw):
    args = pool(kw)
    a = dict(named=P, keep=P, m=2, bs=16)
    a.update(kw)
    _lib.call("fold_free_pages", *args, *a.values(), None, None)


def fork(**kw):
    args = pool(kw)
    import ctypes
    caches = (ctypes.c_int64 * 2)(P, kw.pop("second", P))
    a = dict(src=P, dst=P, m=2, caches=caches, num=2, heads=2, bs=16, row=256, sb=8192, sh=4096, ss=256, ws=P, wb=64)
    a.update(kw)
    _lib.call("fold_fork_pages", *args, *a.values(), None, None)


COMMON = [dict(refs=None), dict(tables=None), dict(lens=None), dict(pages=0), dict(width=-1), dict(rows=-1), dict(stride=3),
          dict(bs=0), dict(m=-1), dict(m=16385)]


@pytest.mark.parametrize("bad", COMMON + [dict(qsl=None), dict(n=-1), dict(pos=None), dict(slots=None),
                                          dict(named=None, m=4), dict(m=16384, width=1 << 18, stride=1 << 18)], ids=str)
def test_grow_refusals(bad):
    with pytest.raises(FoldError, match="grow pages"):
        grow(**bad)


@pytest.mark.parametrize("bad", COMMON + [dict(named=None, m=4)], ids=str)
def test_free_refusals(bad):
    with pytest.raises(FoldError, match="free pages"):
        free(**bad)


@pytest.mark.parametrize("bad", COMMON + [dict(src=None), dict(dst=None), dict(caches=None), dict(second=0), dict(num=-1),
                                          dict(heads=0), dict(row=0), dict(sb=128), dict(sh=255), dict(ss=0), dict(ss=-256),
                                          dict(ws=None), dict(ws=P + 8), dict(wb=32)], ids=str)
def test_fork_refusals(bad):
    with pytest.raises(FoldError, match="fork pages"):
        fork(**bad)


def test_of_nothing_is_a_no_op():
    grow(n=0)
    free(m=0)
    fork(m=0)
    assert _lib.load().fold_fork_pages_workspace(-1) == -1 and _lib.load().fold_fork_pages_workspace(3) > 0


def test_wrappers_take_cuda_tensors_only():
    i, t = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32)
    with pytest.raises(FoldError, match="CUDA"):
        kernels.grow_pages(i, t, i, i, 1, block_size=16)
    with pytest.raises(FoldError, match="CUDA"):
        kernels.free_pages(i, t, i, block_size=16)
    with pytest.raises(FoldError, match="CUDA"):
        kernels.fork_pages(i, t, i, i, i, [torch.zeros(2, 1, 16, 8)])
