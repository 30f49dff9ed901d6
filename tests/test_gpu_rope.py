"""Rotary positions and the paged append on the GPU against the formula in float64."""
import numpy as np
import pytest
import torch

from fold_b200 import kernels, rope
from fold_b200.errors import DEVERR_APPEND_RANGE, DEVERR_ROPE_RANGE, FoldError

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def turned(x, pos, f, interleaved, inverse=False, factor=1.0):
    """(rotated x, error scale of each element) in float64."""
    x = x.double()
    rot = 2 * f.numel()
    ang = pos.double()[:, None] * f.double().to(x.device)
    c, s = (torch.cos(ang) * factor)[:, None], (torch.sin(ang) * factor)[:, None]
    if inverse:
        s = -s
    y, mag = x.clone(), torch.zeros_like(x)
    lo_at = slice(0, rot, 2) if interleaved else slice(0, rot // 2)
    hi_at = slice(1, rot, 2) if interleaved else slice(rot // 2, rot)
    lo, hi = x[..., lo_at], x[..., hi_at]
    y[..., lo_at], y[..., hi_at] = lo * c - hi * s, hi * c + lo * s
    mag[..., lo_at] = mag[..., hi_at] = (lo.abs() + hi.abs()) * factor
    return y, mag


def check(got, want, mag):
    # the table's entries and the two products and the sum round in float32 (2^-24 of the terms
    # each, three in a row), then the result rounds once to its type: half a step of its size
    # (below the normal range, half the smallest step)
    fi = torch.finfo(got.dtype)
    tol = fi.eps / 2 * want.abs() * (1 + 2 ** -20) + 4 * 2 ** -24 * mag + fi.smallest_normal * fi.eps / 2
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


def inputs(n, heads, hd, dt, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(n, heads, hd, generator=g, device="cuda").to(dt)


SHAPES = [  # n, hq, hk, hd, rot
    (1, 1, 1, 64, 64), (1, 32, 8, 128, 128), (5, 7, 1, 80, 32), (3, 4, 2, 96, 24), (17, 3, 3, 128, 30),
    (33, 2, 1, 256, 64), (9, 2, 2, 33, 8), (4, 5, 0, 128, 128), (2100, 16, 4, 128, 128), (700, 9, 2, 64, 32),
    (2, 1, 1, 2, 2)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,hq,hk,hd,rot", SHAPES)
def test_rotary(n, hq, hk, hd, rot, interleaved, dtype):
    x = inputs(n, hq + hk, hd, DT[dtype], n + hd)
    q, k = x[:, :hq], x[:, hq:] if hk else None
    f = rope.default_inv_freq(10000.0, rot)
    table = rope.rope_table(f, 5000, "cuda", factor=1.1)
    pos = torch.randint(0, 5000, (n,), generator=torch.Generator().manual_seed(n)).cuda()
    for inverse in (False, True):
        qo, ko = kernels.rotary(q, k, pos, table, interleaved=interleaved, inverse=inverse)
        check(qo, *turned(q, pos, f, interleaved, inverse, 1.1))
        if hk:
            check(ko, *turned(k, pos, f, interleaved, inverse, 1.1))
        else:
            assert ko is None


def test_rotary_far_positions():
    f = rope.default_inv_freq(500000.0, 128)
    table = rope.rope_table(f, 131072, "cuda")
    pos = torch.tensor([0, 1, 131071, 65537, 99999], device="cuda", dtype=torch.int32)
    q = inputs(5, 4, 128, torch.float32, 3)
    check(kernels.rotary(q, None, pos, table)[0], *turned(q, pos, f, False))


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_in_place_and_strided(interleaved):
    f = rope.default_inv_freq(10000.0, 64)
    table = rope.rope_table(f, 100, "cuda")
    big = inputs(6, 10, 136, torch.bfloat16, 5)
    q = big[:, 1:4, 8:136]  # rows start on 16-byte boundaries
    odd = big[:, 4:7, 3:131]  # rows that do not
    pos = torch.arange(6, device="cuda") * 7
    wants = [turned(x, pos, f, interleaved) for x in (q, odd)]
    rest = big.clone()
    a, b = kernels.rotary(q, None, pos, table, interleaved=interleaved, q_out=q)[0], kernels.rotary(
        odd, None, pos, table, interleaved=interleaved, q_out=odd)[0]
    assert a is q and b is odd
    check(q, *wants[0])
    check(odd, *wants[1])
    rest[:, 1:4, 8:136], rest[:, 4:7, 3:131] = q, odd
    assert torch.equal(rest, big)


@pytest.mark.parametrize("stride", [(128, 1, 1), (1, 1, 1), (0, 128, 1), (256, 0, 1)])
def test_rotary_of_rows_that_share_memory(stride):
    table = rope.rope_table(rope.default_inv_freq(10000.0, 128), 300, "cuda")
    x = inputs(200, 2, 128, torch.bfloat16, 6).as_strided((200, 2, 128), stride)
    pos = torch.arange(200, device="cuda")
    got = kernels.rotary(x, x, pos, table)
    want, _ = kernels.rotary(x.contiguous(), None, pos, table)
    assert torch.equal(got[0], want) and torch.equal(got[1], want)


def test_rotary_inverse_is_the_gradient():
    """The inverse call against differences of a weighted sum of the outputs, and against the
    transpose of the formula."""
    f, c = rope.scaled_inv_freq(10000.0, 32, {"rope_type": "yarn", "factor": 4.0,
                                              "original_max_position_embeddings": 256})
    table = rope.rope_table(f, 1024, "cuda", factor=c)
    x = inputs(5, 2, 48, torch.float32, 1)
    w = inputs(5, 2, 48, torch.float32, 2)
    pos = torch.tensor([3, 0, 1000, 77, 500], device="cuda")
    for inter in (False, True):
        grad, _ = kernels.rotary(w, None, pos, table, interleaved=inter, inverse=True)
        leaf = x.double().requires_grad_(True)
        (turned(leaf, pos, f, inter, False, c)[0] * w.double()).sum().backward()
        check(grad, leaf.grad, w.double().abs().sum(-1, keepdim=True) * c)
        # the map is linear, so a difference of any width is exact up to the rounding of the sums
        for t, h, d in ((0, 1, 0), (2, 0, 31), (4, 1, 47), (3, 0, 16)):
            step = torch.zeros_like(x)
            step[t, h, d] = 1.0
            up, dn = (kernels.rotary(x + s * step, None, pos, table, interleaved=inter)[0].double() for s in (1, -1))
            diff = float(((up - dn) * w.double()).sum() / 2)
            assert abs(diff - float(grad[t, h, d])) <= 64 * 2 ** -24 * float(w.abs().max()) * 8


def test_rotary_reports_positions_outside_the_table():
    table = rope.rope_table(rope.default_inv_freq(10000.0, 64), 50, "cuda")[:50]
    q = inputs(3, 1, 64, torch.bfloat16, 0)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got, _ = kernels.rotary(q, None, torch.tensor([49, 50, -1], device="cuda"), table, err=err)
    assert int(err) == DEVERR_ROPE_RANGE
    want, _ = kernels.rotary(q, None, torch.tensor([49, 49, 0], device="cuda"), table)
    assert torch.equal(got, want)


def cache(nb, hkv, bs, hd, dt, layout, seed=9):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if layout == "heads_first":
        kv = torch.randn(nb, hkv, bs, 2 * hd, generator=g, device="cuda").to(dt)
        return kv, kv[..., :hd], kv[..., hd:]
    kv = torch.randn(2, nb, bs, hkv, hd, generator=g, device="cuda").to(dt)  # slots first, two planes
    return kv, kv[0].transpose(1, 2), kv[1].transpose(1, 2)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("layout", ["heads_first", "slots_first"])
@pytest.mark.parametrize("n,hq,hkv,hd,rot,bs,inter", [
    (1, 32, 8, 128, 128, 16, False), (1, 0, 1, 64, 64, 16, False), (37, 4, 2, 80, 32, 48, True),
    (300, 8, 8, 128, 64, 256, False), (11, 6, 3, 96, 20, 1, True), (5, 2, 1, 7, 4, 3, False),
    (4000, 8, 4, 128, 128, 16, False)])
def test_append_paged(n, hq, hkv, hd, rot, bs, inter, layout, dtype):
    dt = DT[dtype]
    x = inputs(n, hq + 2 * hkv, hd, dt, n)
    q, k, v = x[:, :hq] if hq else None, x[:, hq:hq + hkv], x[:, hq + hkv:]
    nb = -(-n // bs) + 3
    kv, kc, vc = cache(nb, hkv, bs, hd, dt, layout)
    rng = np.random.default_rng(n)
    slots = torch.from_numpy(rng.permutation(nb * bs)[:n]).cuda()
    if n > 3:
        slots[rng.integers(0, n, size=n // 4)] = -1
    f = rope.default_inv_freq(10000.0, rot)
    table = rope.rope_table(f, 4096, "cuda")
    pos = torch.from_numpy(rng.integers(0, 4096, size=n)).cuda()
    want_k, want_v = kc.double().clone(), vc.double().clone()
    mag = torch.zeros_like(want_k)
    live = slots >= 0
    s = slots[live]
    tk, tm = turned(k, pos, f, inter)
    want_k[s // bs, :, s % bs], mag[s // bs, :, s % bs] = tk[live], tm[live]
    want_v[s // bs, :, s % bs] = v.double()[live]
    qo = kernels.append_paged(k, v, pos, slots, kc, vc, table, interleaved=inter, q=q)
    check(kc, want_k, mag)
    assert torch.equal(vc.double(), want_v)
    untouched = mag == 0
    assert torch.equal(kc.double()[untouched], want_k[untouched])  # passed through, or another slot's
    if hq:
        check(qo, *turned(q, pos, f, inter))
    else:
        assert qo is None


def test_append_paged_without_rotation_and_out_of_range():
    k, v = inputs(4, 2, 64, torch.bfloat16, 1), inputs(4, 2, 64, torch.bfloat16, 2)
    kv, kc, vc = cache(2, 2, 16, 64, torch.bfloat16, "heads_first")
    want = kv.clone()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    slots = torch.tensor([5, 32, -7, 31], device="cuda")
    assert kernels.append_paged(k, v, None, slots, kc, vc, None, err=err) is None
    assert int(err) == DEVERR_APPEND_RANGE
    for i, s in ((0, 5), (3, 31)):
        want[s // 16, :, s % 16] = torch.cat([k[i], v[i]], -1)
    assert torch.equal(kv, want)


@pytest.mark.parametrize("n,hq,hkv,hd,rot", [
    (4, 0, 2, 128, 128), (4, 0, 1, 64, 32), (4, 0, 2, 80, 36), (4, 0, 2, 64, 30), (3000, 0, 8, 128, 128),
    (4, 3, 2, 128, 128), (3000, 3, 2, 64, 64), (4, 3, 2, 64, 30)])
def test_positions_of_skipped_tokens(n, hq, hkv, hd, rot):
    """A skipped token's position matters to its query alone: padding rows may hold any position, in
    kernels of wide units (one head a thread, and two) and of a warp a row."""
    x = inputs(n, hq + 2 * hkv, hd, torch.bfloat16, n)
    q, k, v = x[:, :hq] if hq else None, x[:, hq:hq + hkv], x[:, hq + hkv:]
    f = rope.default_inv_freq(10000.0, rot)
    table = rope.rope_table(f, 50, "cuda")[:50]
    kv, kc, vc = cache(-(-n // 16), hkv, 16, hd, torch.bfloat16, "heads_first")
    slots = torch.arange(n, device="cuda")
    slots[1::2] = -1
    pos = torch.arange(n, device="cuda") % 50
    good = pos.clone()
    pos[1::4], pos[3::4], good[1::4], good[3::4] = -1, 50, 0, 49  # as they are clamped
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    want = kv.clone()
    qw = kernels.append_paged(k, v, good, slots, want[..., :hd], want[..., hd:], table, q=q, err=err)
    assert int(err) == 0
    qo = kernels.append_paged(k, v, pos, slots, kc, vc, table, q=q, err=err)
    assert int(err) == (DEVERR_ROPE_RANGE if hq else 0)
    assert torch.equal(kv, want)
    if hq:
        assert torch.equal(qo, qw)


def test_append_paged_offsets_past_32_bits():
    """A cache whose last slots lie past 2^32 elements."""
    nb, hkv, bs, hd = 33000, 8, 64, 128  # 4.3e9 elements, 8.7 GB
    kv = torch.empty(nb, hkv, bs, 2 * hd, dtype=torch.bfloat16, device="cuda")
    last = nb * bs - 1
    kv[-1].zero_()
    k, v = inputs(2, hkv, hd, torch.bfloat16, 1), inputs(2, hkv, hd, torch.bfloat16, 2)
    kernels.append_paged(k, v, None, torch.tensor([last, 0], device="cuda"), kv[..., :hd], kv[..., hd:], None)
    assert torch.equal(kv[-1, :, -1], torch.cat([k[0], v[0]], -1))
    assert torch.equal(kv[0, :, 0], torch.cat([k[1], v[1]], -1))
    assert not bool(kv[-1, :, :-1].any())


def test_in_a_graph_and_on_another_stream():
    f = rope.default_inv_freq(10000.0, 128)
    table = rope.rope_table(f, 4096, "cuda")
    x = inputs(3, 6, 128, torch.bfloat16, 4)
    kv, kc, vc = cache(4, 1, 16, 128, torch.bfloat16, "heads_first")
    pos, slots = torch.tensor([5, 6, 7], device="cuda"), torch.tensor([1, 2, 3], device="cuda")
    out = torch.empty(3, 4, 128, dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kernels.append_paged(x[:, 4:5], x[:, 5:], pos, slots, kc, vc, table, q=x[:, :4], q_out=out)
    torch.cuda.current_stream().wait_stream(side)
    check(out, *turned(x[:, :4], pos, f, False))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kernels.append_paged(x[:, 4:5], x[:, 5:], pos, slots, kc, vc, table, q=x[:, :4], q_out=out)
    pos.copy_(torch.tensor([100, 4000, 9], device="cuda"))
    slots.copy_(torch.tensor([40, -1, 63], device="cuda"))
    kv.zero_()
    g.replay()
    check(out, *turned(x[:, :4], pos, f, False))
    tk, tm = turned(x[:, 4:5], pos, f, False)
    check(kc[2, :, 8], tk[0], tm[0])
    check(kc[3, :, 15], tk[2], tm[2])
    assert torch.count_nonzero(vc).item() == torch.count_nonzero(x[[0, 2], 5]).item()


def test_refusals():
    f = rope.default_inv_freq(10000.0, 64)
    table = rope.rope_table(f, 64, "cuda")
    q = inputs(4, 2, 64, torch.bfloat16, 0)
    pos = torch.arange(4, device="cuda")
    kv, kc, vc = cache(2, 2, 16, 64, torch.bfloat16, "heads_first")
    ok = dict(q_out=None)
    for bad in (lambda: kernels.rotary(q.int(), None, pos, table),
                lambda: kernels.rotary(q, q.float(), pos, table),
                lambda: kernels.rotary(q, q[:2], pos, table),
                lambda: kernels.rotary(q, None, pos[:3], table),
                lambda: kernels.rotary(q, None, pos.float(), table),
                lambda: kernels.rotary(q, None, pos, table.double()),
                lambda: kernels.rotary(q, None, pos, table[:, ::2]),
                lambda: kernels.rotary(q[..., :32], None, pos, table),
                lambda: kernels.rotary(q, None, pos, table, q_out=q[:3]),
                lambda: kernels.rotary(q, None, pos, table, q_out=q.float()),
                lambda: kernels.rotary(q, None, pos, table, err=pos),
                lambda: kernels.append_paged(q, q[:3], pos, pos, kc, vc, table),
                lambda: kernels.append_paged(q, q, pos, pos, kc, vc.contiguous(), table),
                lambda: kernels.append_paged(q.half(), q.half(), pos, pos, kc, vc, table),
                lambda: kernels.append_paged(q, q, pos, pos[:2], kc, vc, table),
                lambda: kernels.append_paged(q, q, pos, pos, kc, vc, None, q=q),
                lambda: kernels.append_paged(q, q, pos, pos, kc, vc, table, q=q[:2])):
        with pytest.raises(FoldError):
            bad()
    e = q[:0]
    out, _ = kernels.rotary(e, None, pos[:0], table, **ok)
    assert out.shape == e.shape
    kernels.append_paged(e, e, pos[:0], pos[:0], kc, vc, table)
