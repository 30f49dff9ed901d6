"""Attention over whole prompts and its gradient on the GPU, against the definition in float64."""
import math

import pytest
import torch

from fold_b200 import kernels, rope
from tests.prompt_cases import DT, FILL, Prompts, check

pytestmark = pytest.mark.gpu


def read(c, causal=True, window=(-1, -1), out=None):
    out = c.full(c.hq) if out is None else out
    lse = torch.full((c.hq, c.n), FILL, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    kernels.prompt_read(c.q, c.k, c.v, c.qsl, out, softmax_scale=c.scale, causal=causal, window_size=window, lse=lse, err=err)
    assert int(err) == 0
    return out, lse


def grad(c, out, lse, causal=True, window=(-1, -1), **kw):
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    g = kernels.prompt_read_grad(c.do, c.q, c.k, c.v, out, lse, c.qsl, softmax_scale=c.scale, causal=causal,
                                 window_size=window, err=err, **kw)
    assert int(err) == 0
    return g


def check_read(c, causal=True, window=(-1, -1)):
    out, lse = read(c, causal, window)
    want, tol = c.oracle(causal, window)
    check(out, want["out"], tol["out"], "out")
    check(lse, want["lse"], tol["lse"], "lse")
    return out, lse


def check_grad(c, causal=True, window=(-1, -1), dlse=None):
    out, lse = read(c, causal, window)
    want, tol = c.oracle(causal, window, dlse)
    rest = c.outside()
    given = [c.full(c.hq), c.full(c.hkv), c.full(c.hkv)]
    grad(c, out, lse, causal, window, dlse=dlse, dq=given[0], dk=given[1], dv=given[2])
    new = grad(c, out, lse, causal, window, dlse=dlse)
    for name, a, b in zip(("dq", "dk", "dv"), given, new):
        check(a, want[name], tol[name], name)  # rows outside hold what they held
        assert torch.equal(a[~rest], b[~rest]) and not bool(b[rest].any())


LENS = [[1], [40], [1, 2, 0, 3, 70], [63, 64, 65], [127, 1, 128, 129], [300, 0, 0, 17], [513]]
HEADS = [(1, 1), (4, 1), (6, 6), (14, 2), (12, 4)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens", LENS, ids=str)
def test_read_lengths(lens, hd, dtype):
    check_read(Prompts(lens, 8, 2, hd, dtype, seed=len(lens) + hd, lead=3, rest=5))


@pytest.mark.parametrize("hd", [8, 72, 80, 96, 136, 192, 248, 256])
@pytest.mark.parametrize("dtype", list(DT))
def test_read_head_sizes(hd, dtype):
    check_read(Prompts([130, 33], 4, 2, hd, dtype, seed=hd, lead=1, rest=2))


@pytest.mark.parametrize("hd", [64, 80, 128])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_read_heads(hq, hkv, hd):
    check_read(Prompts([150, 260], hq, hkv, hd, seed=hq, rest=1))


WINDOWS = [(True, (0, -1)), (True, (1, -1)), (True, (100, -1)), (True, (128, 3)), (False, (-1, -1)), (False, (5, 9)),
           (False, (-1, 130)), (False, (200, 0)), (True, (2000, -1))]


@pytest.mark.parametrize("causal,window", WINDOWS)
@pytest.mark.parametrize("hd", [64, 96, 128])
def test_read_windows(hd, causal, window):
    check_read(Prompts([5, 400, 131], 6, 2, hd, "fp16", seed=hd), causal, window)


@pytest.mark.parametrize("layout", ["packed", "heads_first", "own"])
@pytest.mark.parametrize("hd", [64, 104, 128])
def test_read_layouts(layout, hd):
    c = Prompts([90, 150], 4, 2, hd, layout=layout, seed=3)
    check_read(c)
    # an output inside a wider tensor, and over the queries
    wide = torch.full((c.n, c.hq + 1, hd + 8), FILL, device="cuda", dtype=c.dt)
    want = read(c)[0]
    read(c, out=wide[:, 1:, :hd])
    assert torch.equal(wide[:, 1:, :hd], want) and bool((wide[:, 0] == FILL).all()) and bool((wide[..., hd:] == FILL).all())
    read(c, out=c.q)
    assert torch.equal(c.q, want)


def test_windows_past_every_length():
    c = Prompts([70, 130], 4, 2, 64, seed=4)
    want = read(c, False)[0]
    for window in ((1 << 40, 1 << 33), (-(1 << 40), 1 << 31), (2 ** 31 - 1, 2 ** 30)):
        assert torch.equal(read(c, False, window)[0], want)


def test_read_large_logits():
    for dtype in DT:
        check_read(Prompts([260], 4, 2, 128, dtype, seed=5, boost=6.0))


def test_read_long():
    check_read(Prompts([2200, 900], 2, 1, 128, seed=6))
    check_read(Prompts([2200, 900], 2, 1, 64, seed=6), True, (700, -1))


@pytest.mark.parametrize("hd", [64, 80, 128, 256])
def test_other_sequences_do_not_matter(hd):
    """NaN and infinities of one sequence stay in it, forward and backward."""
    c = Prompts([100, 130, 30], 4, 2, hd, "fp16", seed=hd, layout="own")
    out, lse = read(c)
    g = grad(c, out, lse)
    for x, bad in ((c.q, math.nan), (c.k, math.inf), (c.v, math.nan), (c.do, -math.inf)):
        x[100:230] = bad
    out2, lse2 = read(c)
    rows = torch.ones(260, dtype=torch.bool, device="cuda")
    rows[100:230] = False
    assert torch.equal(out[rows], out2[rows]) and torch.equal(lse[:, rows], lse2[:, rows])
    for a, b in zip(g, grad(c, out2, lse2)):
        assert torch.equal(a[rows], b[rows])


@pytest.mark.parametrize("hd", [64, 80, 128])
def test_nan_reaches_the_outputs(hd):
    c = Prompts([150], 2, 1, hd, seed=1, layout="own")
    c.q[70, 1, 3] = math.nan
    out, lse = read(c)
    assert bool(out[70, 1].isnan().all()) and bool(lse[1, 70].isnan())
    assert int(out.isnan().any(-1).sum()) == 1


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens", LENS, ids=str)
def test_grad_lengths(lens, hd, dtype):
    check_grad(Prompts(lens, 8, 2, hd, dtype, seed=len(lens) + hd, lead=3, rest=5))


@pytest.mark.parametrize("hd", [8, 72, 80, 96, 136, 192, 248, 256])
@pytest.mark.parametrize("dtype", list(DT))
def test_grad_head_sizes(hd, dtype):
    check_grad(Prompts([130, 33], 4, 2, hd, dtype, seed=hd, lead=1, rest=2))


@pytest.mark.parametrize("hd", [64, 80, 128])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_grad_heads(hq, hkv, hd):
    check_grad(Prompts([150, 260], hq, hkv, hd, seed=hq, rest=1))


@pytest.mark.parametrize("causal,window", WINDOWS)
@pytest.mark.parametrize("hd", [64, 96, 128])
def test_grad_windows(hd, causal, window):
    check_grad(Prompts([5, 400, 131], 6, 2, hd, "fp16", seed=hd), causal, window)


@pytest.mark.parametrize("layout", ["packed", "heads_first", "own"])
@pytest.mark.parametrize("hd", [64, 104, 128])
def test_grad_layouts(layout, hd):
    c = Prompts([90, 150], 4, 2, hd, layout=layout, seed=3)
    check_grad(c)
    # gradients side by side in one tensor, as the projection's backward pass takes them
    out, lse = read(c)
    want = grad(c, out, lse)
    x = torch.full((c.n, c.hq + 2 * c.hkv, hd), FILL, device="cuda", dtype=c.dt)
    got = grad(c, out, lse, dq=x[:, :c.hq], dk=x[:, c.hq:c.hq + c.hkv], dv=x[:, c.hq + c.hkv:])
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[0].data_ptr() == x.data_ptr()


@pytest.mark.parametrize("hd", [64, 80, 128])
def test_grad_of_lse(hd):
    c = Prompts([140, 20], 4, 2, hd, seed=9)
    dlse = torch.randn(4, 160, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) * 3
    check_grad(c, dlse=dlse)


@pytest.mark.parametrize("hd", [64, 80, 128])
@pytest.mark.parametrize("lens,window", [([1, 1, 1], (-1, -1)), ([300, 2], (0, 0))])
def test_rows_of_one_key(lens, window, hd):
    """A weight of 1 whatever the logit: queries and keys have no gradient but that of lse."""
    c = Prompts(lens, 4, 2, hd, "fp16", seed=hd)
    out, lse = read(c, True, window)
    dq, dk, dv = grad(c, out, lse, True, window)
    assert not bool(dq.any()) and not bool(dk.any()) and bool(dv.any())
    check_grad(c, True, window, dlse=torch.randn(4, c.n, device="cuda", generator=torch.Generator("cuda").manual_seed(2)))


def test_grad_long():
    check_grad(Prompts([1500, 700], 4, 1, 128, seed=6))
    check_grad(Prompts([1500, 700], 4, 1, 64, seed=6), True, (300, -1))


@pytest.mark.parametrize("hd", [64, 128])
def test_grad_against_differences(hd):
    """Slopes of sum(do o) + sum(dlse lse) by central differences in float64, along random directions."""
    c = Prompts([37, 70], 4, 2, hd, seed=2)
    dlse = torch.randn(4, c.n, device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    out, lse = read(c, True, (50, -1))
    got = dict(zip("qkv", grad(c, out, lse, True, (50, -1), dlse=dlse)))
    _, tol = c.oracle(True, (50, -1), dlse)
    rep = c.hq // c.hkv

    def value(q, k, v):
        total = 0.0
        for i, L in enumerate(c.lens):
            w = slice(c.starts[i], c.starts[i] + L)
            x = torch.einsum("rhd,khd->hrk", q[w], k[w].repeat_interleave(rep, 1)) * c.scale
            d = torch.arange(L, device="cuda")[:, None] - torch.arange(L, device="cuda")[None]
            x = x.masked_fill((d < 0) | (d > 50), -math.inf)
            o = torch.einsum("hrk,khd->rhd", x.softmax(-1), v[w].repeat_interleave(rep, 1))
            total = total + (o * c.do[w].double()).sum() + (torch.logsumexp(x, -1) * dlse[:, w].double()).sum()
        return float(total)

    base = {x: getattr(c, x).double() for x in "qkv"}
    g = torch.Generator("cuda").manual_seed(8)
    for x in "qkv":
        step = torch.randn(base[x].shape, generator=g, device="cuda", dtype=torch.float64)
        h = 1e-5
        up, down = ({**base, x: base[x] + s * h * step} for s in (1, -1))
        slope = (value(**up) - value(**down)) / (2 * h)
        # the difference's own error: rounding of the value by h, and the third derivative, both far below
        bound = float((tol["d" + x] * step.abs()).sum()) + 1e-6 * abs(slope) + 1e-6
        assert abs(float((got[x].double() * step).sum()) - slope) <= bound


def test_equal_calls_give_equal_bits():
    c = Prompts([700, 45, 300], 8, 2, 128, seed=4)
    out, lse = read(c)
    first = grad(c, out, lse)
    for _ in range(3):
        out2, lse2 = read(c)
        assert torch.equal(out, out2) and torch.equal(lse, lse2)
        assert all(torch.equal(a, b) for a, b in zip(first, grad(c, out, lse)))


@pytest.mark.parametrize("hd", [64, 80, 128])
def test_captured_calls_follow_their_lengths(hd):
    """One graph of forward and backward, replayed with other lengths and inputs."""
    a, b = Prompts([100, 160], 4, 2, hd, seed=1, layout="own"), Prompts([1, 200], 4, 2, hd, seed=2, layout="own", rest=59)
    out, lse = a.full(4), torch.full((4, 260), FILL, device="cuda")
    g = [a.full(4), a.full(2), a.full(2)]
    ws = kernels.prompt_grad_workspace(260, 4, 2, hd, "cuda")

    def step():
        kernels.prompt_read(a.q, a.k, a.v, a.qsl, out, softmax_scale=a.scale, lse=lse)
        kernels.prompt_read_grad(a.do, a.q, a.k, a.v, out, lse, a.qsl, softmax_scale=a.scale, dq=g[0], dk=g[1], dv=g[2],
                                 workspace=ws)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for c in (a, b):
        for name in ("q", "k", "v", "do", "qsl"):
            getattr(a, name).copy_(getattr(c, name))
        for x in (out, lse, *g):
            x.fill_(FILL)
        graph.replay()
        want, tol = c.oracle()
        for name, x in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *g)):
            check(x, want[name], tol[name], name)


def test_two_calls_at_once():
    cs = [Prompts([400, 77 + i], 4, 2, 128, seed=i) for i in range(4)]
    want = []
    for c in cs:
        o, l = read(c)
        want.append((o, l, *grad(c, o, l)))
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    got = []
    for c, s in zip(cs, streams):
        with torch.cuda.stream(s):
            out, lse = torch.empty_like(want[0][0][:c.n]), torch.empty((4, c.n), device="cuda")
            out = torch.empty((c.n, 4, 128), device="cuda", dtype=c.dt)
            kernels.prompt_read(c.q, c.k, c.v, c.qsl, out, softmax_scale=c.scale, lse=lse)
            got.append((out, lse, *kernels.prompt_read_grad(c.do, c.q, c.k, c.v, out, lse, c.qsl, softmax_scale=c.scale)))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_many_short_sequences():
    lens = [(i * 7) % 12 for i in range(300)]
    c = Prompts(lens, 4, 2, 64, seed=11, rest=3)
    check_read(c)
    check_grad(c)


def test_nothing():
    c = Prompts([5], 2, 1, 64)
    out = c.full(2)
    kernels.prompt_read(c.q, c.k, c.v, c.qsl[:1], out, softmax_scale=1.0)
    assert bool((out == FILL).all())
    lse = torch.zeros(2, 5, device="cuda")
    assert not any(bool(x.any()) for x in kernels.prompt_read_grad(c.do, c.q, c.k, c.v, out, lse, c.qsl[:1], softmax_scale=1.0))
    kernels.prompt_read(c.q[:0], c.k[:0], c.v[:0], c.qsl[:1], out[:0], softmax_scale=1.0)


def test_prompt_to_cache_and_back():
    """The path in order: rotary, attention over the prompts, append, the cache's read of the same rows, the
    gradient turned back through the rotation."""
    hq, hkv, hd, bs = 8, 2, 128, 16
    c = Prompts([70, 33], hq, hkv, hd, seed=21, layout="own")
    n = c.n
    table = rope.rope_table(rope.scaled_inv_freq(10000.0, hd, None)[0].cuda(), 4096, "cuda")
    refs = torch.zeros(20, dtype=torch.int32, device="cuda")
    tables, lens = torch.zeros((2, 8), dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    positions, slots = kernels.grow_pages(refs, tables, lens, c.qsl, n, block_size=bs)
    assert positions.tolist() == list(range(70)) + list(range(33))
    raw = c.q, c.k
    c.q, c.k = kernels.rotary(c.q, c.k, positions, table)
    out, lse = check_read(c)
    kv = torch.full((20, hkv, bs, 2 * hd), math.nan, device="cuda", dtype=c.dt)
    kc, vc = kernels.paged_planes(kv, hd)
    kernels.append_paged(raw[1], c.v, positions, slots, kc, vc, table)
    again, lse2 = torch.empty_like(out), torch.empty_like(lse)
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    kernels.prefix_read(c.q, c.qsl, lens, none, kc, vc, none, tables, again, softmax_scale=c.scale, lse=lse2)
    want, tol = c.oracle()
    check(again, want["out"], tol["out"], "the cache's read")
    dq, dk, dv = grad(c, out, lse)
    check(dq, want["dq"], tol["dq"], "dq")
    dq0, dk0 = kernels.rotary(dq, dk, positions, table, inverse=True)
    # a rotation keeps the size of every pair; turned forward again it is the gradient up to two roundings
    dq1, _ = kernels.rotary(dq0, None, positions, table)
    err = (dq1.double() - dq.double()).abs()
    pair = torch.hypot(dq.double()[..., :hd // 2], dq.double()[..., hd // 2:]).repeat(1, 1, 2)
    assert bool((err <= 3 * c.u * pair + 2.0 ** -24).all())
    assert dk0.shape == dk.shape and bool(torch.isfinite(dv).all())
