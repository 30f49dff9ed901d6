"""Refusals of the attention over whole prompts and its gradient that need no GPU."""
import pytest
import torch

from fold_b200 import _lib, kernels
from fold_b200.errors import FoldError


def read(**kw):
    a = dict(q=16, qs=(512, 128), k=32, ks=(256, 128), v=48, vs=(256, 128), qsl=16, b=1, left=-1, right=-1, scale=1.0,
             out=64, os=(512, 128), n=2, hq=4, hkv=2, hd=128, dtype=0)
    a.update(kw)
    _lib.call("fold_prompt_read", a["q"], *a["qs"], a["k"], *a["ks"], a["v"], *a["vs"], a["qsl"], a["b"], 1, a["left"],
              a["right"], a["scale"], a["out"], *a["os"], None, a["n"], a["hq"], a["hkv"], a["hd"], a["dtype"], None, None)


def grad(**kw):
    a = dict(do=64, dos=(512, 128), q=16, qs=(512, 128), k=32, ks=(256, 128), v=48, vs=(256, 128), o=80, os=(512, 128),
             lse=16, qsl=16, b=1, scale=1.0, dq=96, dqs=(512, 128), dk=112, dks=(256, 128), dv=128, dvs=(256, 128), ws=16,
             wb=1 << 30, n=2, hq=4, hkv=2, hd=128, dtype=0, rest=1)
    a.update(kw)
    _lib.call("fold_prompt_read_grad", a["do"], *a["dos"], a["q"], *a["qs"], a["k"], *a["ks"], a["v"], *a["vs"], a["o"],
              *a["os"], a["lse"], None, a["qsl"], a["b"], 1, -1, -1, a["scale"], a["dq"], *a["dqs"], a["dk"], *a["dks"],
              a["dv"], *a["dvs"], a["rest"], a["ws"], a["wb"], a["n"], a["hq"], a["hkv"], a["hd"], a["dtype"], None, None)


SIZES = [dict(n=-1), dict(b=-1), dict(hq=3), dict(hq=0), dict(hkv=0), dict(hd=0), dict(hd=12), dict(hd=264),
         dict(dtype=2), dict(dtype=7), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")),
         dict(qsl=None), dict(q=None), dict(k=None), dict(v=None), dict(q=8), dict(k=24), dict(v=4), dict(qs=(508, 128)),
         dict(ks=(256, 124)), dict(vs=(-256, 128)), dict(hq=1 << 17, hkv=1), dict(n=(1 << 30) + 1)]


@pytest.mark.parametrize("bad", SIZES + [dict(out=None), dict(out=8), dict(os=(0, 128)), dict(os=(512, 0)),
                                         dict(os=(256, 128)), dict(os=(512, 64)), dict(os=(-512, 128)),
                                         dict(out=32), dict(out=48)], ids=str)
def test_read_refusals(bad):
    with pytest.raises(FoldError, match="prompt read"):
        read(**bad)


@pytest.mark.parametrize("bad", SIZES + [dict(do=None), dict(o=None), dict(lse=None), dict(dq=None), dict(dk=None),
                                         dict(dv=None), dict(dqs=(128, 128)), dict(dks=(256, 64)), dict(dvs=(0, 128)),
                                         dict(ws=None), dict(wb=8), dict(ws=24), dict(do=2), dict(b=0),
                                         dict(dq=16), dict(dk=32), dict(dv=112), dict(dk=80), dict(dv=64)], ids=str)
def test_grad_refusals(bad):
    with pytest.raises(FoldError, match="prompt read grad"):
        grad(**bad)


def test_of_nothing_is_a_no_op():
    read(n=0)
    read(b=0)
    grad(n=0)
    grad(b=0, rest=0)


def test_workspace_sizes():
    assert 0 < _lib.prompt_read_grad_workspace(1, 32, 8, 128) < _lib.prompt_read_grad_workspace(4096, 32, 8, 128)
    for bad in ((-1, 8, 8, 128), (1, 8, 3, 128), (1, 0, 1, 128), (1, 8, 8, 100), (1, 8, 8, 512)):
        assert _lib.prompt_read_grad_workspace(*bad) == -1


def test_wrappers_check_what_they_get():
    x, qsl = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(FoldError, match="CUDA"):
        kernels.prompt_read(x, x, x, qsl, x, softmax_scale=1.0)
    with pytest.raises(FoldError, match="CUDA"):
        kernels.prompt_read_grad(x, x, x, x, x, torch.zeros(2, 3), qsl, softmax_scale=1.0)
    with pytest.raises(FoldError, match="CUDA"):
        kernels.prompt_grad_workspace(1, 1, 1, 64, "cpu")
