"""Attention over whole prompts and its gradient where every block takes several items of several tiles, against float64."""
import math
import random

import pytest
import torch

from tests.prompt_cases import DT, Prompts, check
from tests.test_gpu_prompt import grad, read

pytestmark = pytest.mark.gpu

# Sequences, their least and most rows, heads. With the SMs' 148 blocks an item is followed by others, keys' and
# rows': 24 sequences of 2 KV heads split a group of four into its heads, 12 of 8 KV heads into pairs; where a
# device's blocks have three key tiles each (tiles x KV heads >= 444) an item has all heads of its group.
PACKS = [(24, 100, 700, 8, 2), (12, 100, 700, 32, 8), (7, 150, 550, 64, 32), (17, 60, 600, 48, 16)]


def pack(shape, hd, dtype, layout="packed"):
    b, lo, hi, hq, hkv = shape
    rng = random.Random(b + hd)
    lens = [rng.randint(lo, hi) for _ in range(b)]
    lens[1], lens[3] = 1, 0
    return Prompts(lens, hq, hkv, hd, dtype, seed=b + hd, lead=2, rest=3, layout=layout)


def compare(c, causal=True, window=(-1, -1), dlse=None, rows=slice(None)):
    """Forward and backward, at the given rows; the backward pass three times with equal bits."""
    out, lse = read(c, causal, window)
    want, tol = c.oracle(causal, window, dlse)
    check(out[rows], want["out"][rows], tol["out"][rows], "out")
    check(lse[:, rows], want["lse"][:, rows], tol["lse"][:, rows], "lse")
    first = None
    for _ in range(3):
        got = [c.full(c.hq), c.full(c.hkv), c.full(c.hkv)]
        grad(c, out, lse, causal, window, dlse=dlse, dq=got[0], dk=got[1], dv=got[2])
        got = [x[rows] for x in got]
        first = first or got
        for name, x, y in zip(("dq", "dk", "dv"), got, first):
            check(x, want[name][rows], tol[name][rows], name)
            assert torch.equal(x, y), f"{name} has other bits in another call"


@pytest.mark.parametrize("causal,window", [(True, (-1, -1)), (True, (200, -1)), (False, (90, 150))])
@pytest.mark.parametrize("hd", [64, 80, 128])
@pytest.mark.parametrize("shape", PACKS, ids=str)
def test_items_behind_items(shape, hd, causal, window):
    """Accumulators, tiles and places that one item leaves are the next one's."""
    dtype = "fp16" if hd == 80 or window[1] > 0 else "bf16"
    c = pack(shape, hd, dtype)
    dlse = torch.randn(c.hq, c.n, device="cuda", generator=torch.Generator("cuda").manual_seed(7)) if window[0] > 0 else None
    compare(c, causal, window, dlse)


@pytest.mark.parametrize("window", [(-1, -1), (130, -1)])
@pytest.mark.parametrize("hd", [64, 128])
def test_neighbours_of_cut_tiles(hd, window):
    """Tiles cut in either half, beside sequences of NaN and infinities: weights of zero meet zeros."""
    for hq, hkv in ((8, 2), (10, 2)):
        lens = [x for i in range(40) for x in (128 * (i % 4) + 3 * i + 1, 140)]
        c = Prompts(lens, hq, hkv, hd, "bf16", seed=hd, layout="own", rest=130)
        rows = torch.ones(c.n, dtype=torch.bool, device="cuda")
        for i in range(1, len(lens), 2):
            w = slice(c.starts[i], c.starts[i + 1])
            rows[w] = False
            for x, bad in ((c.q, math.nan), (c.k, math.inf), (c.v, -math.inf), (c.do, math.nan)):
                x[w] = bad
        rows[c.starts[-1]:] = False
        compare(c, True, window, rows=rows)


@pytest.mark.parametrize("first", [False, True])
def test_results_beside_the_inputs(first):
    """Outputs that are views of the inputs' tensor, tokens or heads first, and share no row with them."""
    n, hq, hkv, hd = 200, 4, 2, 64
    c = Prompts([150, 50], hq, hkv, hd, seed=3, layout="own")
    out, lse = read(c)
    want = grad(c, out, lse)
    heads = [hq, hkv, hkv, hq, hq, hkv, hkv]
    x = torch.zeros((sum(heads), n, hd) if first else (n, sum(heads), hd), device="cuda", dtype=c.dt)
    parts = [p.transpose(0, 1) if first else p for p in x.split(heads, 0 if first else 1)]
    for p, t in zip(parts, (c.q, c.k, c.v)):
        p.copy_(t)
    c.q, c.k, c.v = parts[:3]
    assert torch.equal(read(c, out=parts[3])[0], out)
    got = grad(c, parts[3], lse, dq=parts[4], dk=parts[5], dv=parts[6])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
