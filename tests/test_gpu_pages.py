"""Pages of a paged cache on the GPU (grow, fork, free), against the same steps on the host."""
import math
import random

import pytest
import torch

from fold_b200 import kernels
from fold_b200.errors import (DEVERR_BLOCK_TABLE, DEVERR_CAPACITY, DEVERR_PAGES, DEVERR_REFS, DEVERR_ROW,
                              DEVERR_SHARED, FoldError)

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Pool:
    """The pool on the device and the same on the host: page lists in place of tables and counts."""

    def __init__(self, pages, rows, width, bs):
        self.pages, self.width, self.bs = pages, width, bs
        self.refs, self.lens = ints([0] * pages), ints([0] * rows)
        self.tables = torch.full((rows, width), -7, dtype=torch.int32, device="cuda")
        self.err = ints([0])
        self.held, self.tokens = [[] for _ in range(rows)], [0] * rows

    def counts(self):
        c = [0] * self.pages
        for h in self.held:
            for p in h:
                c[p] += 1
        return c

    def free_list(self):
        return [p for p, c in enumerate(self.counts()) if c == 0]

    def need(self, tokens):
        return -(-tokens // self.bs)

    def check(self, err=0):
        assert int(self.err) == err
        self.err.zero_()
        assert self.lens.tolist() == self.tokens
        assert self.refs.tolist() == self.counts()
        t = self.tables.tolist()
        for r, h in enumerate(self.held):
            assert t[r][:len(h)] == h, r

    def grow(self, add, rows=None, spare=0, lead=0, err=0):
        starts = [lead]
        for a in add:
            starts.append(starts[-1] + a)
        n = starts[-1] + spare
        pos, slots = kernels.grow_pages(self.refs, self.tables, self.lens, ints(starts), n, block_size=self.bs,
                                        rows=None if rows is None else ints(rows), err=self.err)
        free, short, seen = self.free_list(), False, set()
        counts = self.counts()
        want_pos, want_slots = [0] * n, [-1] * n
        for i, a in enumerate(add):
            r = i if rows is None else rows[i]
            if r < 0 or r >= len(self.tokens) or r in seen:
                continue
            seen.add(r)
            old = self.tokens[r]
            if old + a > self.width * self.bs or (a and old % self.bs and counts[self.held[r][-1]] > 1):
                continue
            k = self.need(old + a) - self.need(old)
            if k and (short or k > len(free)):
                short = True
                continue
            self.held[r] = self.held[r] + free[:k]
            free = free[k:]
            self.tokens[r] = old + a
            for x in range(a):
                want_pos[starts[i] + x] = old + x
                want_slots[starts[i] + x] = self.held[r][(old + x) // self.bs] * self.bs + (old + x) % self.bs
        self.check(err)
        assert slots.tolist() == want_slots
        assert [p for p, s in zip(pos.tolist(), want_slots) if s >= 0] == [p for p, s in zip(want_pos, want_slots) if s >= 0]
        return pos, slots

    def free(self, rows=None, keep=None, err=0):
        kernels.free_pages(self.refs, self.tables, self.lens, None if rows is None else ints(rows), block_size=self.bs,
                           keep=None if keep is None else ints(keep), err=self.err)
        for i, r in enumerate(range(len(self.tokens)) if rows is None else rows):
            if 0 <= r < len(self.tokens):
                self.tokens[r] = min(self.tokens[r], max(0 if keep is None else keep[i], 0))
                self.held[r] = self.held[r][:self.need(self.tokens[r])]
        self.check(err)

    def fork(self, src, dst, caches, err=0):
        before = [c.clone() for c in caches]
        kernels.fork_pages(self.refs, self.tables, self.lens, ints(src), ints(dst), caches, err=self.err)
        free, counts = self.free_list(), self.counts()
        seen, was, tokens, short = set(), [list(h) for h in self.held], list(self.tokens), False
        for s, d in zip(src, dst):
            if s < 0 or d < 0 or max(s, d) >= len(tokens) or tokens[d] or d in seen:
                continue
            seen.add(d)
            t = tokens[s]
            if t % self.bs:
                if not free:
                    continue
                page = free.pop(0)
                for c, b in zip(caches, before):
                    b[page][:, :t % self.bs] = b[was[s][-1]][:, :t % self.bs]
                self.held[d] = was[s][:t // self.bs] + [page]
            else:
                self.held[d] = list(was[s])
            self.tokens[d] = t
        self.check(err)
        for c, b in zip(caches, before):
            assert torch.equal(c.view(torch.uint8), b.view(torch.uint8))


def cache(pages, heads, bs, width, layers=1, dtype=torch.bfloat16, layout="heads_first"):
    g = torch.Generator("cuda").manual_seed(pages)
    out = []
    for _ in range(layers):
        shape = (pages, heads, bs, width) if layout == "heads_first" else (pages, bs, heads, width)
        x = torch.randn(shape, generator=g, device="cuda").to(dtype)
        out.append(x if layout == "heads_first" else x.transpose(1, 2))
    return out


@pytest.mark.parametrize("bs", [1, 16, 48])
def test_grow(bs):
    p = Pool(200, 6, 40, bs)
    p.grow([5, 0, 1, bs, 2 * bs + 1, 17], spare=3)
    p.grow([1] * 6)
    p.grow([bs - 1, 3 * bs], rows=[5, 0], lead=2)
    p.grow([0] * 6)


def test_grow_takes_the_lowest_free_pages():
    p = Pool(60, 4, 20, 16)
    p.grow([100, 100, 100, 100])
    p.free([1, 3], [20, 0])
    p.grow([64, 70, 16, 90])
    assert p.held[0][7:] == [9, 10, 11, 12][:len(p.held[0][7:])]


def test_grow_in_a_large_pool_and_of_many_sequences():
    p = Pool(70001, 1500, 60, 16)
    rng = random.Random(1)
    p.grow([rng.randint(0, 700) for _ in range(1500)])
    rows = rng.sample(range(1500), 1300)
    p.free(rows, [rng.randint(0, 300) for _ in rows])
    rows = rng.sample(range(1500), 1100)
    p.grow([rng.randint(0, 12) for _ in rows], rows=rows, spare=9, lead=3)


def test_refusals_among_many_tokens():
    p = Pool(120, 6, 40, 16)
    p.grow([500, 641, 500, 640, 3, 300], spare=5, err=DEVERR_CAPACITY | DEVERR_PAGES)  # too long; no pages for the last
    assert p.tokens == [500, 0, 500, 640, 3, 0]
    p.grow([600, 600, 7], rows=[4, 1, 4], lead=1, err=DEVERR_ROW | DEVERR_PAGES)


def test_grow_of_the_most_sequences():
    m = 16384
    p = Pool(17000, m, 2, 4)
    p.grow([1] * m)
    p.grow([3] * m, rows=list(range(m - 1, -1, -1)))
    with pytest.raises(FoldError, match="16384"):
        kernels.grow_pages(p.refs, p.tables, p.lens, ints([0] * (m + 2)), 1, block_size=4, rows=ints([0] * (m + 1)))


def test_grow_without_pages():
    p = Pool(10, 5, 8, 16)
    p.grow([40, 16, 16 * 7, 1, 0], err=DEVERR_PAGES)  # 3 + 1 pages, then seven do not fit: the next is not served either
    assert p.tokens == [40, 16, 0, 0, 0]
    p.grow([8, 0, 0, 0, 3])  # no new page for the first
    p.grow([1, 0, 0, 95, 0], err=DEVERR_PAGES)
    p.grow([0, 0, 16 * 4, 0, 0])
    p.grow([0, 0, 1, 0, 0], err=DEVERR_PAGES)


def test_grow_refusals():
    p = Pool(50, 4, 3, 16)
    p.grow([10, 49, 48, 0], err=DEVERR_CAPACITY)
    p.grow([1, 2, 3], rows=[0, 0, 3], err=DEVERR_ROW)  # named twice: the first
    p.grow([5, 5, 5], rows=[-1, 9, 1], err=DEVERR_ROW)
    p.grow([2, 2, 1], rows=[-1, -1, 3])
    p.fork([0], [1], [cache(50, 1, 16, 8)[0]], err=DEVERR_ROW)  # row 1 is in use


def test_shared_partly_filled_page_does_not_grow():
    p = Pool(20, 3, 4, 16)
    kv = cache(20, 1, 16, 8)
    p.grow([40, 0, 0])
    p.fork([0], [1], kv)
    p.free([1], [20])             # into the second page, which both hold
    p.grow([0, 1, 0], err=DEVERR_SHARED)
    p.fork([1], [2], kv)          # a fork may be written
    p.grow([0, 0, 12])
    p.free([0])
    p.grow([0, 1, 0])             # and so may the last one that holds it


@pytest.mark.parametrize("dtype,width,layout", [(torch.bfloat16, 256, "heads_first"), (torch.float16, 80, "tokens_first"),
                                                (torch.float32, 6, "heads_first"), (torch.float16, 3, "heads_first"),
                                                (torch.uint8, 7, "tokens_first")])
def test_fork_copies(dtype, width, layout):
    p = Pool(64, 9, 8, 16)
    kv = cache(64, 3, 16, width, 3, dtype if dtype.is_floating_point else torch.float32, layout)
    kv = [x if dtype.is_floating_point else (x * 50).to(torch.uint8) for x in kv]
    p.grow([33, 16, 1, 100, 0, 0, 0, 0, 0])
    p.fork([0, 0, 3, 1], [4, 6, 5, 8], kv)
    p.fork([2, -1, 5], [7, 2, -1], kv)


def test_fork_of_planes_and_many_layers():
    kv = cache(30, 2, 16, 32, 200)
    planes = [x[..., :16] for x in kv] + [x[..., 16:] for x in kv]
    p = Pool(30, 4, 8, 16)
    p.grow([45, 0, 0, 0])
    p.fork([0, 0], [1, 3], planes)


def test_fork_refusals():
    p = Pool(6, 6, 8, 16)
    kv = cache(6, 1, 16, 8)
    p.grow([20, 33, 0, 0, 0, 0])
    p.fork([0, 1, 0], [2, 2, 9], kv, err=DEVERR_ROW)      # the same child twice: the first; no such row
    p.fork([0, 1], [3, 4], kv, err=DEVERR_PAGES)          # no page left: the children stay empty
    p.fork([0, 4, 3], [1, 5, 3], kv, err=DEVERR_ROW)      # row 1 is in use; empty parents
    p.free([1])
    p.fork([2, 2], [3, 4], kv)


def test_free():
    p = Pool(64, 8, 8, 16)
    kv = cache(64, 1, 16, 8)
    p.grow([100, 33, 7, 0, 16, 0, 0, 0])
    p.fork([0, 0, 1], [5, 6, 7], kv)
    p.free([0, 0, 1, -1], [50, 20, 200, 0])       # a row twice: the smaller length
    p.free([5, 5, 2])
    p.free([3, 11], err=DEVERR_ROW)
    p.free(None, [0, 1, 2, 3, 4, 5, 6, -8])
    p.free()
    assert not bool(p.refs.any())


def test_bad_tables_are_reported():
    p = Pool(8, 3, 4, 16)
    p.grow([40, 0, 0])
    p.tables[0, 1] = 99
    kernels.free_pages(p.refs, p.tables, p.lens, ints([0]), block_size=16, err=p.err)
    assert int(p.err) == DEVERR_BLOCK_TABLE and p.refs.tolist() == [0, 1] + [0] * 6
    p.err.zero_()
    p.lens[1], p.tables[1, 0] = 10, 5            # a page that nobody holds
    kernels.free_pages(p.refs, p.tables, p.lens, ints([1]), block_size=16, err=p.err)
    assert int(p.err) == DEVERR_REFS and p.refs.tolist() == [0, 1] + [0] * 6
    p.err.zero_()
    p.lens[2] = 1 << 20
    kernels.grow_pages(p.refs, p.tables, p.lens, ints([0, 0, 0, 2]), 2, block_size=16, err=p.err)
    assert int(p.err) == DEVERR_CAPACITY and int(p.lens[2]) == 1 << 20


def test_a_long_run_of_steps():
    rng = random.Random(5)
    p = Pool(120, 12, 30, 16)
    kv = cache(120, 2, 16, 16, 2)
    p.grow([60, 100, 5, 31] + [0] * 8)
    for _ in range(60):
        live = [r for r, t in enumerate(p.tokens) if t]
        empty = [r for r, t in enumerate(p.tokens) if not t]
        what = rng.random()
        if what < 0.4 and live:
            rows = rng.sample(live, rng.randint(1, len(live)))
            old = [p.tokens[r] for r in rows]
            add = [rng.randint(0, 9) for _ in rows]
            shared = any(a and t % 16 and p.counts()[p.held[r][-1]] > 1 for a, t, r in zip(add, old, rows))
            need = sum(p.need(t + a) - p.need(t) for a, t in zip(add, old))
            if not shared and need <= len(p.free_list()) and max(old) < 400:
                p.grow(add, rows=rows)
                p.free(rows, [t + rng.randint(0, a) for t, a in zip(old, add)])
        elif what < 0.7 and live and empty:
            dst = rng.sample(empty, rng.randint(1, min(3, len(empty))))
            if len(p.free_list()) >= len(dst):
                p.fork([rng.choice(live) for _ in dst], dst, kv)
        elif live and len(live) > 3:
            p.free(rng.sample(live, rng.randint(1, 2)))


def test_captured_step():
    """Grow and trim in one graph, replayed behind other lengths."""
    p = Pool(100, 4, 20, 16)
    p.grow([30, 40, 50, 0])
    qsl, keep = ints([0, 5, 10, 15, 20]), p.lens.clone()
    pos, slots = torch.zeros(20, dtype=torch.int64, device="cuda"), torch.zeros(20, dtype=torch.int64, device="cuda")

    def step():
        kernels.grow_pages(p.refs, p.tables, p.lens, qsl, 20, block_size=16, positions=pos, slots=slots, err=p.err)
        kernels.free_pages(p.refs, p.tables, p.lens, block_size=16, keep=keep, err=p.err)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    graph.replay()
    p.check()
    first = pos.tolist()
    p.grow([2, 2, 2, 2])
    keep.copy_(p.lens)
    graph.replay()
    p.check()
    assert pos.tolist() == [x + 2 for x in first]


def test_forked_sequences_read_as_their_parent():
    """A prompt appended, forked, each child grown by its own tokens: the cache's read against float64."""
    hq, hkv, hd, bs, n0, c = 4, 2, 64, 16, 37, 3
    g = torch.Generator("cuda").manual_seed(3)
    p = Pool(40, 1 + c, 8, bs)
    kv = torch.full((40, hkv, bs, 2 * hd), math.nan, device="cuda", dtype=torch.float16)
    kc, vc = kernels.paged_planes(kv, hd)

    def tokens(n):
        return (torch.randn(n, hkv, hd, generator=g, device="cuda").half() for _ in range(2))

    k0, v0 = tokens(n0)
    pos, slots = p.grow([n0, 0, 0, 0])
    kernels.append_paged(k0, v0, None, slots, kc, vc, None)
    p.fork([0] * c, [1, 2, 3], [kv.nan_to_num_(0.5)])
    k1, v1 = tokens(2 * c)
    pos, slots = p.grow([2] * c, rows=[1, 2, 3])
    assert pos.tolist() == [n0, n0 + 1] * c
    kernels.append_paged(k1, v1, None, slots, kc, vc, None)
    q = torch.randn(2 * c, hq, hd, generator=g, device="cuda").half()
    out, none = torch.empty_like(q), ints([0])
    kernels.prefix_read(q, ints([0, 2, 4, 6]), p.lens[1:].contiguous(), none, kc, vc, none, p.tables[1:], out,
                        softmax_scale=hd ** -0.5)
    for i in range(c):
        k, v = (torch.cat([a, b[2 * i:2 * i + 2]]).double().repeat_interleave(2, 1) for a, b in ((k0, k1), (v0, v1)))
        x = torch.einsum("rhd,khd->hrk", q[2 * i:2 * i + 2].double(), k) * hd ** -0.5
        x[:, 0, n0 + 1] = -math.inf
        w = x.softmax(-1)
        want = torch.einsum("hrk,khd->rhd", w, v)
        size = torch.einsum("hrk,khd->rhd", w, v.abs())
        # weights and result round once to fp16 (2^-11 each), logits in float32: far below one more of them
        assert bool(((out[2 * i:2 * i + 2].double() - want).abs() <= 2.0 ** -11 * (2 * size + want.abs())).all())
