"""The gradient of the prompts' attention against central differences of the attention itself, in float64, along
directions in which a wrong gradient shows: a part along the gradient, so that slopes do not cancel."""
import math

import pytest
import torch

from tests.prompt_cases import Prompts
from tests.test_gpu_prompt import grad, read

pytestmark = pytest.mark.gpu


def value(c, q, k, v, dlse, causal, window):
    """sum(do o) + sum(dlse lse)."""
    total = 0.0
    for i, L in enumerate(c.lens):
        w = slice(c.starts[i], c.starts[i] + L)
        rep = c.hq // c.hkv
        x = torch.einsum("rhd,khd->hrk", q[w], k[w].repeat_interleave(rep, 1)) * c.scale
        d = torch.arange(L, device="cuda")[:, None] - torch.arange(L, device="cuda")[None]
        hidden = torch.zeros_like(d, dtype=torch.bool)
        if causal:
            hidden |= d < 0
        if window[0] >= 0:
            hidden |= d > window[0]
        if window[1] >= 0:
            hidden |= -d > window[1]
        x = x.masked_fill(hidden, -math.inf)
        o = torch.einsum("hrk,khd->rhd", x.softmax(-1), v[w].repeat_interleave(rep, 1))
        total = total + (o * c.do[w].double()).sum() + (torch.logsumexp(x, -1) * dlse[:, w].double()).sum()
    return float(total)


@pytest.mark.parametrize("causal,window", [(True, (-1, -1)), (True, (50, -1)), (False, (20, 31))])
@pytest.mark.parametrize("hd", [64, 96, 128, 192])
def test_slopes(hd, causal, window):
    c = Prompts([37, 170], 4, 2, hd, "fp16", seed=2)
    dlse = torch.randn(4, c.n, device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    out, lse = read(c, causal, window)
    got = dict(zip("qkv", grad(c, out, lse, causal, window, dlse=dlse)))
    want, _ = c.oracle(causal, window, dlse)
    base = {x: getattr(c, x).double() for x in "qkv"}
    g = torch.Generator("cuda").manual_seed(8)
    for x in "qkv":
        exact, kernel = want["d" + x], got[x].double()
        # the kernel's error is a few roundings of fp16 (2^-11 each) of the gradient, in the norm; along one direction
        # no more than that, and a quarter of a hundredth is five such roundings
        size = float(exact.norm())
        assert float((kernel - exact).norm()) <= size / 400
        for _ in range(3):
            step = torch.randn(base[x].shape, generator=g, device="cuda", dtype=torch.float64)
            step = exact / size + step / step.norm()
            step /= step.norm()
            h = 1e-5
            up, down = ({**base, x: base[x] + s * h * step} for s in (1, -1))
            slope = (value(c, **up, dlse=dlse, causal=causal, window=window)
                     - value(c, **down, dlse=dlse, causal=causal, window=window)) / (2 * h)
            # the difference's own error: the value's rounding (2^-53 of some 10^5) by h, and h^2 times its third
            # derivative along a step of length 1
            assert abs(float((exact * step).sum()) - slope) <= 1e-6 * abs(slope) + 1e-6
            off = lambda gradient: abs(float((gradient * step).sum()) - slope)  # noqa: E731
            assert off(kernel) <= size / 400
            assert off(0 * kernel) > size / 10 and off(-kernel) > size / 10 and off(kernel * 1.02) > size / 400
