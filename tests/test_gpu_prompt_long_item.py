"""A KV head's tile that passes thousands of heads' rows takes longer than a wait may last."""
import pytest
import torch

from fold_b200 import kernels

pytestmark = pytest.mark.gpu


def test_item_of_seconds():
    """4000 heads of 56832 rows on one KV head: 2.7 s for the first tile of keys. Rows lie over one another (inputs may),
    so that only dq takes memory."""
    n, hq, hd = 56832, 4000, 64
    g = torch.Generator("cuda").manual_seed(0)
    x = torch.randn(n * 8 + hq * 64 + 64, device="cuda", generator=g).to(torch.bfloat16).as_strided((n, hq, hd), (8, 64, 1))
    k, v = (torch.randn(n, 1, hd, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    lse = torch.full((hq, n), 12.0, device="cuda")
    qsl = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    dq, dk, dv = kernels.prompt_read_grad(x, x, k, v, x, lse, qsl, softmax_scale=hd ** -0.5, err=err)
    assert int(err) == 0
    assert bool(torch.isfinite(dk).all()) and bool(torch.isfinite(dv).all())
    # the last key is seen by the last row of every head alone
    q = x[-1].double()
    p = torch.exp((q * hd ** -0.5) @ k[-1, 0].double() - 12.0)
    want = (p[:, None] * q).sum(0)
    bound = (p[:, None] * q.abs()).sum(0) * 2.0 ** -8 * 1.1 + want.abs() * 2.0 ** -8 + 1e-30  # P's rounding, the result's
    assert bool(((dv[-1, 0].double() - want).abs() <= bound).all())
