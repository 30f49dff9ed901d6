"""How exact the prompts' attention and its gradient are, in the norm, against float64.

Bounds on single elements add up the worst of every rounding and pass a kernel that lost half of its bits. Here the
roundings that a kernel may make are made in float64 and their effects added as independent errors are (their norms by
squares), so that one more rounding than those shows:

  every result      its own rounding to the type
  out, dv           P, rounded once: P's last bits, whatever its size
  dq, dk            delta from the out that it was given (rows of more than 8 keys), and, where a row sees many keys,
                    dS rounded once, whatever its size
"""
import math

import pytest
import torch

from tests.prompt_cases import DT, Prompts
from tests.test_gpu_prompt import grad, read

pytestmark = pytest.mark.gpu

# The products' float32 sums are a hundredth of a rounding of fp16 (4096 / 16 steps of 2^-24, at random, to 2^-11), and
# two samples of the same roundings over 40000 elements have norms within a hundredth; the rest is room.
ROOM = 1.05


def rounded(x, dt):
    """x with as many bits as the type has, of any size."""
    m, e = torch.frexp(x)
    bits = 8 if dt is torch.bfloat16 else 11
    return torch.ldexp(torch.round(m * 2.0 ** bits), e - bits)


def errors(c, out, causal, window):
    """Results in float64 and the norms that their errors may have."""
    hq, hkv, hd, s = c.hq, c.hkv, c.hd, c.scale
    g = hq // hkv
    parts = {k: [] for k in ("out", "dq", "dk", "dv")}
    total = {k: 0.0 for k in parts}
    for i, L in enumerate(c.lens):
        w = slice(c.starts[i], c.starts[i] + L)
        q, do, o16 = (x[w].double().transpose(0, 1) for x in (c.q, c.do, out))
        k, v = (x[w].double().transpose(0, 1).repeat_interleave(g, 0) for x in (c.k, c.v))
        d = torch.arange(L, device="cuda")[:, None] - torch.arange(L, device="cuda")[None]
        seen = (d >= 0) if causal else torch.ones_like(d, dtype=torch.bool)
        if window[0] >= 0:
            seen = seen & (d <= window[0])
        count, row = seen.sum(1), torch.arange(L, device="cuda")
        p = ((q * s) @ k.transpose(1, 2)).masked_fill_(~seen, -math.inf).softmax(2)
        dp_p = rounded(p, c.dt) - p
        o = p @ v
        off = ((do * (o16 - o)).sum(2) * (count > 8))[..., None] * p       # of dS, by delta
        ds = p * (do @ v.transpose(1, 2) - (do * o).sum(2, keepdim=True))
        # rows of few keys have dS in two parts, and those behind a window of up to 2048
        once = (count > 512) & ~((window[0] >= 0) & (window[0] < 2048) & (row > window[0] + 127))
        ds_p = (rounded(ds, c.dt) - ds) * once[:, None]

        def by_key(t):
            return t.reshape(hkv, g, L, hd).sum(1)

        effects = {"out": [dp_p @ v], "dv": [by_key(dp_p.transpose(1, 2) @ do)],
                   "dq": [s * (x @ k) for x in (off, ds_p)], "dk": [by_key(s * (x.transpose(1, 2) @ q)) for x in (off, ds_p)]}
        for name, x in (("out", o), ("dv", by_key(p.transpose(1, 2) @ do)), ("dq", s * (ds @ k)),
                        ("dk", by_key(s * (ds.transpose(1, 2) @ q)))):
            parts[name].append(x.transpose(0, 1))
            total[name] += float(((x.to(c.dt).double() - x) ** 2).sum()) + sum(float((y ** 2).sum()) for y in effects[name])
    return {k: torch.cat(x) for k, x in parts.items()}, {k: math.sqrt(x) for k, x in total.items()}


def compare(c, causal=True, window=(-1, -1)):
    out, lse = read(c, causal, window)
    want, norm = errors(c, out, causal, window)
    got = dict(zip(("out", "dq", "dk", "dv"), (out, *grad(c, out, lse, causal, window))))
    ratio = {k: float((got[k].double() - want[k]).norm()) / norm[k] for k in got}
    assert max(ratio.values()) <= ROOM, ratio


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("hd", [64, 80, 128, 256])
@pytest.mark.parametrize("lens", [[2] * 60, [3] * 60, [6, 5, 4] * 20, [8] * 40, [9, 20] * 20], ids=lambda x: str(x[:3]))
def test_few_tokens(lens, hd, dtype):
    compare(Prompts(lens, 8, 2, hd, dtype, seed=len(lens)))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("lens,causal,window", [([100, 300, 200], True, (-1, -1)), ([511], False, (-1, -1)),
                                                ([2600], True, (100, -1)), ([2600], True, (511, -1)),
                                                ([3100], True, (2047, -1)), ([2500], True, (-1, -1))])
def test_longer_rows(lens, causal, window, hd, dtype):
    compare(Prompts(lens, 4, 2, hd, dtype, seed=hd), causal, window)


@pytest.mark.parametrize("size", [100.0, 1.0, 1e-2, 1e-3, 1e-4])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n,causal", [(4096, True), (3000, False), (300, True)])
def test_small_gradients(n, causal, hd, size):
    """A gradient that a mean over many tokens leaves: dS of thousands of keys is far below the smallest normal number
    of fp16 where dq and dk are not."""
    c = Prompts([n], 4, 2, hd, "fp16", seed=hd)
    c.do = (c.do.float() * size).to(c.dt)
    compare(c, causal)


@pytest.mark.parametrize("hd", [64, 256])
def test_gradients_of_different_sizes(hd):
    """One sequence's large gradient does not take the bits of another's, nor do rows without one."""
    c = Prompts([700, 900, 1000], 4, 2, hd, "fp16", seed=hd)
    size = torch.ones(c.n, 1, 1, device="cuda")
    size[:700], size[700:1600], size[1000:1400] = 300.0, 1e-3, 0.0
    c.do = (c.do.float() * size).to(c.dt)
    out, lse = read(c)
    got = grad(c, out, lse)
    for i, L in enumerate(c.lens):
        w = slice(c.starts[i], c.starts[i] + L)
        one = Prompts([L], 4, 2, hd, "fp16")
        one.q, one.k, one.v, one.do = c.q[w], c.k[w], c.v[w], c.do[w]
        want, norm = errors(one, out[w], True, (-1, -1))
        ratio = {k: float((x[w].double() - want[k]).norm()) / norm[k] for k, x in zip(("dq", "dk", "dv"), got)}
        assert max(ratio.values()) <= ROOM, (i, ratio)
