"""Refusals of fold_prefix_read that need no GPU."""
import pytest
import torch

from fold_b200 import _lib, kernels
from fold_b200.errors import FoldError


def call(**kw):
    a = dict(q=16, qs=(512, 128), qsl=16, own=16, plen=16, b=1, k=16, v=16 + 256, nb=4, bs=16, cs=(8192, 4096, 256),
             pt=16, ptl=2, bt=16, bts=2, btl=2, out=16, os=(512, 128), ws=16, wb=1 << 40, n=2, hq=4, hkv=2, hd=128,
             dtype=0)
    a.update(kw)
    _lib.call("fold_prefix_read", a["q"], *a["qs"], a["qsl"], a["own"], a["plen"], a["b"], a["k"], a["v"], a["nb"],
              a["bs"], *a["cs"], a["pt"], a["ptl"], a["bt"], a["bts"], a["btl"], 1, 1.0, a["out"], *a["os"], None,
              a["ws"], a["wb"], a["n"], a["hq"], a["hkv"], a["hd"], a["dtype"], None, None)


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(qsl=None), dict(own=None), dict(plen=None), dict(k=None), dict(v=None), dict(pt=None),
    dict(bt=None), dict(out=None), dict(n=-1), dict(b=-1), dict(hq=3), dict(hq=0), dict(hkv=0), dict(nb=0),
    dict(bs=0), dict(bs=8), dict(bs=24), dict(ptl=-1), dict(btl=-1), dict(hd=96), dict(hd=0), dict(dtype=2),
    dict(dtype=9), dict(hq=129 * 2), dict(q=8), dict(k=24), dict(v=8), dict(out=4), dict(qs=(512, 4)),
    dict(os=(508, 128)), dict(cs=(8192, 4096, 260)), dict(cs=(8192 + 8, 4096, 256)), dict(ws=None), dict(wb=16),
    dict(ws=8), dict(nb=1 << 31), dict(os=(0, 128)), dict(os=(512, 0))])
def test_refusals(bad):
    with pytest.raises(FoldError, match="prefix read"):
        call(**bad)


@pytest.mark.parametrize("strides", [(0, 128), (512, 0), (512, 120), (64, 128), (512, -8)])
def test_output_rows_that_share_memory_are_refused(strides):
    with pytest.raises(FoldError, match="share memory"):
        call(os=strides)


def test_of_nothing_is_a_no_op():
    call(n=0)
    call(b=0)


def test_workspace_sizes():
    small = _lib.prefix_read_workspace(1, 32, 8, 128)
    large = _lib.prefix_read_workspace(4096, 32, 8, 128)
    assert 0 < small < large
    for bad in ((-1, 8, 8, 128), (1, 8, 3, 128), (1, 0, 1, 128), (1, 8, 8, 96), (1, 256, 1, 128)):
        assert _lib.prefix_read_workspace(*bad) == -1


def test_wrapper_takes_cuda_tensors_only():
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    kv = torch.zeros(2, 1, 16, 128, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(FoldError, match="CUDA"):
        kernels.prefix_read(x, torch.zeros(2, dtype=torch.int32), i, i, kv[..., :64], kv[..., 64:], i, i[None], x,
                            softmax_scale=1.0)
