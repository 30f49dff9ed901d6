"""The shared-prefix read on the GPU against the definition in float64."""
import math

import numpy as np
import pytest
import torch

from fold_b200 import kernels, rope
from fold_b200.errors import DEVERR_BLOCK_TABLE, DEVERR_CAPACITY, FoldError

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


class Case:
    """A paged cache with shuffled blocks, every slot that no length reaches filled with NaN."""

    def __init__(self, nq, own, prefix, hq, hkv, hd, bs, dtype="bf16", seed=0, layout="heads_first", boost=1.0,
                 spare_rows=0, table_pad=2):
        rng = np.random.default_rng(seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        dt = DT[dtype]
        self.nq, self.own, self.prefix, self.hkv, self.hd, self.bs = nq, own, prefix, hkv, hd, bs
        n = sum(nq) + spare_rows
        self.q = (torch.randn(n, hq, hd, generator=g, device="cuda") * boost).to(dt)
        pb, ob = -(-prefix // bs), [-(-o // bs) for o in own]
        nb = pb + sum(ob) + 2
        perm = rng.permutation(nb).astype(np.int32)
        if layout == "heads_first":
            kv = torch.full((nb, hkv, bs, 2 * hd), math.nan, device="cuda", dtype=dt)
            self.k, self.v = kv[..., :hd], kv[..., hd:]
        else:
            kv = torch.full((2, nb, bs, hkv, hd), math.nan, device="cuda", dtype=dt)
            self.k, self.v = kv[0].transpose(1, 2), kv[1].transpose(1, 2)
        self.kv = kv

        def fill(blocks, length):
            k = torch.randn(length, hkv, hd, generator=g, device="cuda")
            k[..., rng.integers(0, hd)] *= 4.0
            v = torch.randn(length, hkv, hd, generator=g, device="cuda")
            v[..., rng.integers(0, hd)] *= 8.0
            k, v = k.to(dt), v.to(dt)
            j = np.arange(length)
            blk, off = torch.from_numpy(blocks[j // bs].astype(np.int64)).cuda(), torch.from_numpy(j % bs).cuda()
            self.k[blk, :, off], self.v[blk, :, off] = k, v
            return k, v

        self.parts = [fill(perm[:pb], prefix)]
        tables = np.full((len(nq), max(ob + [0]) + table_pad), nb + 5, dtype=np.int32)  # unused entries: no block
        at = pb
        for i, m in enumerate(ob):
            tables[i, :m] = perm[at:at + m]
            self.parts.append(fill(perm[at:at + m], own[i]))
            at += m
        self.prefix_table = torch.from_numpy(np.concatenate([perm[:pb], np.full(1, -3, np.int32)])).cuda()
        self.tables = torch.from_numpy(tables).cuda()
        self.qsl = torch.tensor(np.concatenate([[0], np.cumsum(nq)]), dtype=torch.int32, device="cuda")
        self.own_lens = torch.tensor(own, dtype=torch.int32, device="cuda")
        self.prefix_len = torch.tensor([prefix], dtype=torch.int32, device="cuda")
        self.scale = hd ** -0.5

    def args(self):
        return (self.q, self.qsl, self.own_lens, self.prefix_len, self.k, self.v, self.prefix_table, self.tables)

    def read(self, causal=True, **kw):
        out = torch.full(self.q.shape, 77.0, device="cuda", dtype=self.q.dtype)
        lse = torch.full((self.q.shape[1], self.q.shape[0]), 77.0, device="cuda")
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        kernels.prefix_read(*self.args(), out, softmax_scale=self.scale, causal=causal, lse=lse, err=err, **kw)
        assert int(err) == 0
        return out, lse

    def oracle(self, causal=True):
        """(out, lse, tolerance of out, tolerance of lse) in float64."""
        n, hq, hd = self.q.shape
        u = torch.finfo(self.q.dtype).eps / 2
        out = torch.full((n, hq, hd), 77.0, dtype=torch.float64, device="cuda")
        lse = torch.full((hq, n), 77.0, dtype=torch.float64, device="cuda")
        tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
        pk, pv = self.parts[0]
        a = 0
        for i, rows in enumerate(self.nq):
            ok, ov = self.parts[1 + i]
            k, v = torch.cat([pk, ok]).double(), torch.cat([pv, ov]).double()
            L, m = k.shape[0], self.own[i]
            seen = torch.ones(rows, L, dtype=torch.bool, device="cuda")
            if causal:
                last = m - rows + torch.arange(rows, device="cuda")
                seen[:, self.prefix:] = torch.arange(m, device="cuda")[None] <= last[:, None]
            for h in range(hq):
                kh, vh = k[:, h // (hq // self.hkv)], v[:, h // (hq // self.hkv)]
                qh = self.q[a:a + rows, h].double() * self.scale
                x = (qh @ kh.T).masked_fill(~seen, -math.inf)
                z = torch.logsumexp(x, 1) if L else torch.full((rows,), -math.inf, dtype=torch.float64, device="cuda")
                p = torch.exp(x - torch.where(torch.isinf(z), 0.0, z)[:, None])
                o, A = p @ vh, p @ vh.abs()
                # float32 logits: hd + 2 roundings of the terms' sizes (2^-23: the accumulation may
                # truncate); exp2 and the running rescales a few units in 2^-22 more
                mag = (qh.abs() @ kh.abs().T).masked_fill(~seen, 0.0).amax(1) if L else torch.zeros_like(z)
                ex = (hd + 2) * 2.0 ** -23 * mag + 2.0 ** -19
                # weights and result round once to the type (u each); products accumulate in float32
                acc = (L / 16 + 64) * 2.0 ** -23
                tol[a:a + rows, h] = (u + 2 * ex + acc)[:, None] * A * 1.01 + u * o.abs() + 2.0 ** -24
                out[a:a + rows, h], lse[h, a:a + rows] = o, z
                ltol[h, a:a + rows] = 2 * ex + acc + 2.0 ** -22 * torch.where(torch.isinf(z), 0.0, z).abs()
            a += rows
        return out, lse, tol, ltol

    def check(self, causal=True, **kw):
        out, lse = self.read(causal, **kw)
        wo, wl, tol, ltol = self.oracle(causal)
        err = (out.double() - wo).abs()
        assert bool(torch.isfinite(out).all())
        assert bool((err <= tol).all()), f"out off by {float((err - tol).max())} past its tolerance"
        same = torch.isinf(wl) & torch.isinf(lse)
        lerr = torch.where(same, 0.0, (lse.double() - wl).abs())
        assert bool((lerr <= ltol).all()), f"lse off by {float((lerr - ltol).max())} past its tolerance"
        return out, lse


HEADS = [(4, 1), (8, 8), (14, 2), (5, 1), (32, 8)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_decode(hq, hkv, hd, dtype):
    Case([1, 1, 1, 1], [1, 130, 17, 255], 300, hq, hkv, hd, 16, dtype, seed=hd + hq).check()


@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 127, 128, 129, 256, 1000])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prefix_lengths(hd, prefix):
    Case([1, 2, 3], [1, 2, 40], prefix, 8, 2, hd, 16, seed=prefix).check()


@pytest.mark.parametrize("bs", [16, 32, 48, 64, 80, 128, 256, 384])
@pytest.mark.parametrize("layout", ["heads_first", "slots_first"])
def test_blocks_and_layouts(bs, layout):
    Case([3, 1, 2], [200, 1, 385], 517, 8, 2, 128, bs, seed=bs, layout=layout).check()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hd,hq,hkv", [(64, 6, 2), (128, 8, 2), (256, 4, 2), (128, 7, 1)])
def test_ragged_rows(hd, hq, hkv, causal):
    """Row counts around the tiles' borders, rows without keys, sequences without rows."""
    nq = [1, 0, 5, 64, 33, 130, 0, 2, 9]
    own = [0, 7, 5, 64, 200, 131, 0, 1, 3]  # [2]: none past its rows; [7], [8]: rows before the first key
    Case(nq, own, 70, hq, hkv, hd, 16, seed=hd).check(causal)
    Case(nq, own, 0, hq, hkv, hd, 16, seed=hd).check(causal)


@pytest.mark.parametrize("hq,hkv", [(64, 2), (128, 1), (17, 1), (96, 2), (24, 1)])
def test_wide_groups(hq, hkv):
    """Groups of many heads: one token fills a row tile, or three fill half of one."""
    Case([1, 3, 2, 9], [40, 3, 200, 9], 260, hq, hkv, 128, 16, seed=hq).check()
    Case([1, 5], [1, 300], 0, hq, hkv, 64, 32, "fp16", seed=hq).check()


def test_output_in_place_of_the_query():
    c = Case([1, 4, 70], [30, 200, 70], 300, 8, 2, 128, 16)
    want, _ = c.check()
    kernels.prefix_read(*c.args(), c.q, softmax_scale=c.scale)
    assert torch.equal(c.q, want)


def test_broadcast_query_heads():
    """A query whose heads share memory is read as if it were copied out."""
    c = Case([1, 2], [30, 60], 100, 8, 2, 128, 16)
    c.q = c.q[:, :1].expand(3, 8, 128)
    out = torch.empty(3, 8, 128, device="cuda", dtype=torch.bfloat16)
    kernels.prefix_read(*c.args(), out, softmax_scale=c.scale)
    c.q = c.q.contiguous()
    assert torch.equal(out, c.read()[0])


def test_blocks_past_32_bits():
    """Keys in blocks that lie past 2^32 elements of the cache."""
    nb, hkv, bs, hd = 33000, 8, 64, 128
    kv = torch.empty(nb, hkv, bs, 2 * hd, dtype=torch.bfloat16, device="cuda")
    c = Case([1, 20], [100, 150], 200, 8, 8, 128, 64, seed=3)
    used = c.kv.shape[0]
    kv[-used:] = c.kv
    c.k, c.v = kv[..., :hd], kv[..., hd:]
    shift = nb - used
    c.prefix_table += shift
    c.tables += shift
    c.check()


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_workspace_on_any_16_byte_boundary(hd):
    """A workspace cut out of a larger buffer, at every 16-byte boundary of a sector, for segments of
    few and of many rows; nothing beside it is written."""
    c = Case([1, 30, 3], [70, 300, 3], 500, 8, 2, hd, 16, seed=hd)
    want, wl = c.check()
    size = kernels.prefix_workspace(34, 8, 2, hd, "cuda").numel()
    arena = torch.empty(size + 256, device="cuda", dtype=torch.uint8)
    assert arena.data_ptr() % 32 == 0
    for at in (0, 16, 32, 48, 112):
        arena.fill_(171)
        out, lse = c.read(workspace=arena[at:at + size])
        assert torch.equal(out, want) and torch.equal(lse, wl)
        assert bool((arena[:at] == 171).all()) and bool((arena[at + size:] == 171).all())


def test_rows_that_see_nothing():
    c = Case([2, 1, 3], [0, 0, 1], 0, 4, 2, 128, 16)
    out, lse = c.check()
    assert not bool(out[:5].any()) and bool(torch.isinf(lse[:, :5]).all())
    assert bool(torch.isfinite(lse[:, 5]).all())


@pytest.mark.parametrize("own,prefix", [([40, 9], 0), ([0, 0], 300), ([0, 0], 0)])
def test_tables_of_no_blocks(own, prefix):
    c = Case([2, 1], own, prefix, 8, 2, 128, 16, table_pad=0)
    c.prefix_table = c.prefix_table[:-(-prefix // 16)]
    assert c.prefix_table.numel() == 0 or prefix
    c.check(causal=False)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_long_split(hd):
    """Few rows over many keys (split over the SMs and joined), and one long sequence among short."""
    Case([1], [3], 20011, 4, 1, hd, 16, seed=1).check()
    Case([1, 1, 2], [9000, 5, 40], 100, 4, 2, hd, 64, seed=2).check()


@pytest.mark.parametrize("dtype", list(DT))
def test_many_rows(dtype):
    Case([1] * 150, list(np.random.default_rng(0).integers(1, 300, 150)), 1500, 8, 2, 128, 16, dtype, seed=3).check()
    Case([700, 300], [900, 300], 600, 4, 2, 128, 32, dtype, seed=4).check()


def test_many_sequences():
    rng = np.random.default_rng(5)
    Case([int(x) for x in rng.integers(0, 3, 1000)], [int(x) for x in rng.integers(0, 40, 1000)], 33, 2, 1, 64, 16,
         seed=5).check()


@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("tiles", [1, 2, 5, 14, 30, 61, 100])
def test_short_pieces_of_a_wide_prefix(tiles, hd):
    """Few units in all: every piece is as short as pieces get, about one wide key tile."""
    Case([1] * 40 + [24], [3] * 40 + [24], 128 * tiles - 5, 4, 1, hd, 16, seed=tiles).check()


@pytest.mark.parametrize("prefix", [700, 2048, 3333])
@pytest.mark.parametrize("hd", [64, 128])
def test_line_cut_where_few_rows_begin(hd, prefix):
    """Many-row items of the prefix and few-row items of the sequences, both over dozens of CTAs."""
    rng = np.random.default_rng(prefix)
    Case([1] * 210, rng.integers(1, 200, 210).tolist(), prefix, 8, 2, hd, 16, seed=prefix).check()


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_many_short_parts_between_long_ones(hd):
    """Row tiles of every width behind one another in one launch: sequences of one token, of a few
    and of hundreds, with many short parts between the long ones."""
    rng = np.random.default_rng(hd)
    nq, own = [], []
    for i in range(120):
        nq.append(int(rng.choice([1, 1, 1, 1, 2, 5, 9, 33, 40, 70, 130])))
        own.append(int(rng.choice([0, 1, 60, 130, 400])) if i % 3 else 128 + nq[-1])
    Case(nq, own, 300, 8, 2, hd, 16, seed=hd).check()
    Case(nq, own, 0, 4, 4, hd, 32, "fp16", seed=hd).check(causal=False)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_stale_slots_behind_every_long_segment(hd):
    """Segments of many rows that each end inside a page of scattered small pages, tile counts of
    one to seven in turn: the last tile's stale slots (NaN) are zeroed while tiles before it may
    still be on their way through the ring. Every pass gives the same bits."""
    rng = np.random.default_rng(hd)
    nq = [20 + int(x) for x in rng.integers(0, 60, 96)]
    own = [max(n, 128 * (i % 7) + 1 + int(rng.integers(0, 127))) for i, n in enumerate(nq)]
    c = Case(nq, own, 0, 4, 4, hd, 16, seed=hd)
    want, wl = c.check()
    for _ in range(20):
        out, lse = c.read()
        assert torch.equal(out, want) and torch.equal(lse, wl)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_large_logits(hd, dtype):
    """Logits of some hundreds: rows whose mass sits on single keys and whose maximum rises often."""
    Case([1, 4], [300, 900], 700, 4, 2, hd, 16, dtype, seed=6, boost=30.0).check()


def test_rising_maxima():
    """Keys that grow along the prefix, so that every tile raises every row's maximum."""
    c = Case([1, 8], [64, 64], 2000, 4, 2, 128, 16, seed=7)
    k = c.parts[0][0]
    j = torch.arange(2000, device="cuda")
    ramp = (c.q[0, 0].float() * (j[:, None].float() / 60.0) * 128 ** -0.5 / 8).to(torch.bfloat16)
    k.copy_(ramp[:, None].expand_as(k))
    blk = c.prefix_table.long()[j // 16]
    c.k[blk, :, j % 16] = k
    c.check()


def test_rows_behind_the_last_sequence_are_left():
    c = Case([2, 3], [10, 20], 50, 8, 2, 128, 16, spare_rows=4)
    out, lse = c.check()  # the oracle keeps the 77s there
    assert bool((out[5:] == 77).all()) and bool((lse[:, 5:] == 77).all())


def test_strides():
    c = Case([2, 1], [30, 200], 140, 8, 2, 128, 16)
    want, wl = c.check()
    big = torch.zeros(3, 16, 256, dtype=torch.bfloat16, device="cuda")
    big[:, 2:10, 64:192] = c.q
    c.q = big[:, 2:10, 64:192]
    wide = torch.full((3, 9, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    out = wide[:, 1:]
    kernels.prefix_read(*c.args(), out, softmax_scale=c.scale)
    assert torch.equal(out, want) and bool((wide[:, 0] == 5).all())
    tab = torch.zeros(2, 50, dtype=torch.int32, device="cuda")
    tab[:, :c.tables.shape[1]] = c.tables
    c.tables = tab[:, :c.tables.shape[1]]
    assert torch.equal(c.read()[0], want)
    c.q = c.q.transpose(1, 2).contiguous().transpose(1, 2)  # heads not contiguous: copied
    assert torch.equal(c.read()[0], want)


def test_bad_tables_and_lengths_are_reported():
    c = Case([1, 2], [30, 60], 100, 4, 2, 128, 16)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.empty_like(c.q)
    good = c.tables.clone()
    c.tables[1, 1] = -1
    kernels.prefix_read(*c.args(), out, softmax_scale=c.scale, err=err)
    assert int(err) == DEVERR_BLOCK_TABLE and bool(torch.isfinite(out).all())
    # the missing block reads as zeros
    c.tables = good
    blk = int(good[1, 1])
    c.kv[blk] = 0
    assert torch.equal(c.read()[0], out)
    err.zero_()
    c.own_lens[0] = 1 << 20
    kernels.prefix_read(*c.args(), out, softmax_scale=c.scale, err=err)
    assert int(err) & DEVERR_CAPACITY


def test_deterministic_graph_and_streams():
    c = Case([1, 3, 2], [700, 20, 333], 3000, 8, 2, 128, 16, seed=8)
    want, wl = c.check()
    for _ in range(3):
        out, lse = c.read()
        assert torch.equal(out, want) and torch.equal(lse, wl)
    # two streams at once, each with a workspace of its own
    outs = [torch.empty_like(c.q) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s, o in zip(streams, outs):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(5):
                kernels.prefix_read(*c.args(), o, softmax_scale=c.scale)
    for s, o in zip(streams, outs):
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(o, want)
    # captured once, replayed at other lengths
    ws = kernels.prefix_workspace(c.q.shape[0], 8, 2, 128, "cuda")
    out = torch.empty_like(c.q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kernels.prefix_read(*c.args(), out, softmax_scale=c.scale, workspace=ws)
    g.replay()
    assert torch.equal(out, want)
    c.prefix_len.copy_(torch.tensor([1234]))
    c.own_lens.copy_(torch.tensor([11, 0, 333]))
    c.qsl.copy_(torch.tensor([0, 3, 3, 6]))
    g.replay()
    again = torch.empty_like(out)
    kernels.prefix_read(*c.args(), again, softmax_scale=c.scale)
    assert torch.equal(out, again)
    c.nq, c.own, c.prefix = [3, 0, 3], [11, 0, 333], 1234
    c.parts[0] = tuple(x[:1234] for x in c.parts[0])
    c.parts[1:] = [tuple(x[:m] for x in part) for part, m in zip(c.parts[1:], c.own)]
    c.check()


def test_rotate_append_and_read_together():
    """The three operators as a serving step uses them: prompt and step tokens rotated and stored,
    then read, against float64 attention over float64-rotated keys."""
    hq, hkv, hd, bs, prefix, b = 8, 2, 128, 16, 333, 3
    f, c = rope.scaled_inv_freq(10000.0, hd, {"rope_type": "yarn", "factor": 4.0,
                                              "original_max_position_embeddings": 512})
    table = rope.rope_table(f, 4096, "cuda", factor=c)
    g = torch.Generator(device="cuda").manual_seed(0)
    kv = torch.full((60, hkv, bs, 2 * hd), math.nan, device="cuda", dtype=torch.float16)
    kc, vc = kernels.paged_planes(kv, hd)
    ids = torch.randperm(60, generator=g, device="cuda").to(torch.int32)
    ptab, tabs = ids[:21].contiguous(), ids[21:21 + 9].view(3, 3).contiguous()
    pk = torch.randn(prefix, 2 * hkv, hd, generator=g, device="cuda").half()
    j = torch.arange(prefix, device="cuda")
    kernels.append_paged(pk[:, :hkv], pk[:, hkv:], j, ptab[j // bs].long() * bs + j % bs, kc, vc, table)
    own = [1, 20, 37]
    rows = [1, 3, 2]
    pos, slot, toks = [], [], []
    for i in range(b):
        o = torch.arange(own[i], device="cuda")
        pos.append(prefix + o)
        slot.append(tabs[i][o // bs].long() * bs + o % bs)
        toks.append(torch.randn(own[i], hq + 2 * hkv, hd, generator=g, device="cuda").half())
    x = torch.cat(toks)
    q = kernels.append_paged(x[:, hq:hq + hkv], x[:, hq + hkv:], torch.cat(pos), torch.cat(slot), kc, vc, table,
                             q=x[:, :hq])
    sel = torch.cat([torch.arange(sum(own[:i + 1]) - rows[i], sum(own[:i + 1])) for i in range(b)]).cuda()
    q = q[sel].contiguous()
    out = torch.empty_like(q)
    kernels.prefix_read(q, torch.tensor([0, 1, 4, 6], dtype=torch.int32, device="cuda"),
                        torch.tensor(own, dtype=torch.int32, device="cuda"),
                        torch.tensor([prefix], dtype=torch.int32, device="cuda"), kc, vc, ptab, tabs, out,
                        softmax_scale=hd ** -0.5)

    def rot(t, p):
        ang = p.double()[:, None] * f.double().cuda()
        cs, sn = (torch.cos(ang) * c)[:, None], (torch.sin(ang) * c)[:, None]
        lo, hi = t.double()[..., :hd // 2], t.double()[..., hd // 2:]
        return torch.cat([lo * cs - hi * sn, hi * cs + lo * sn], -1)

    at, r = 0, 0
    for i in range(b):
        k = torch.cat([rot(pk[:, :hkv], j), rot(toks[i][:, hq:hq + hkv], pos[i])])
        v = torch.cat([pk[:, hkv:], toks[i][:, hq + hkv:]]).double()
        qi = rot(toks[i][own[i] - rows[i]:, :hq], pos[i][own[i] - rows[i]:])
        for t in range(rows[i]):
            L = prefix + own[i] - rows[i] + t + 1
            for h in range(hq):
                kh, vh = k[:L, h // 4], v[:L, h // 4]
                logit = kh @ qi[t, h] * hd ** -0.5
                p = torch.softmax(logit, 0)
                # q and k each round to fp16 (2^-11 of every product's size), the weights and the
                # result once more
                d = 2 * 2.0 ** -11 * float((kh.abs() @ qi[t, h].abs()).max()) * hd ** -0.5
                tol = (2 * d + 2.0 ** -11 + 2.0 ** -12) * (p @ vh.abs()) + 2.0 ** -11 * (p @ vh).abs()
                assert bool(((out[r, h].double() - p @ vh).abs() <= tol).all())
            r += 1
        at += own[i]


def test_refusals():
    c = Case([1, 2], [30, 60], 100, 4, 2, 128, 16)
    out = torch.empty_like(c.q)
    q, qsl, own, plen, k, v, pt, bt = c.args()

    def bad(*a, o=out, **kw):
        with pytest.raises(FoldError):
            kernels.prefix_read(*a, o, softmax_scale=1.0, **kw)

    bad(q.float(), qsl, own, plen, k, v, pt, bt, o=out.float())
    bad(q.half(), qsl, own, plen, k, v, pt, bt, o=out.half())
    bad(q, qsl[:2], own, plen, k, v, pt, bt)
    bad(q, qsl.long(), own, plen, k, v, pt, bt)
    bad(q, qsl, own, plen.long(), k, v, pt, bt)
    bad(q, qsl, own, plen, k, v.contiguous(), pt, bt)
    bad(q, qsl, own, plen, k, v, pt, bt[:1])
    bad(q, qsl, own, plen, k, v, pt, bt.t())
    bad(q, qsl, own, plen, k, v, pt, bt, o=out[:2])
    bad(q, qsl, own, plen, k, v, pt, bt, lse=torch.empty(3, 4, device="cuda"))
    bad(q, qsl, own, plen, k, v, pt, bt, workspace=torch.empty(16, device="cuda", dtype=torch.uint8))
    bad(q[..., :64], qsl, own, plen, k, v, pt, bt, o=out[..., :64])
    bad(q, qsl, own, plen, k, v, pt, bt, err=own.float())
    kernels.prefix_read(q[:0], torch.zeros(3, dtype=torch.int32, device="cuda"), own, plen, k, v, pt, bt, out[:0],
                        softmax_scale=1.0)
