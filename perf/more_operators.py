"""Operators around the paged path and the sizes they are measured at.

Each in a plain form (elementary torch operations in 32 bits) and as the calls a user makes of
fold_b200.kernels:

  prompt_read       attention over whole prompts: sequences of different lengths packed one behind the
                    other, causal, heads in groups that share keys and values, a sliding window
  prompt_read_grad  its gradient: those of queries, keys and values from that of the output
  fork_pages        sequences of a paged cache forked: full pages shared, a partly filled last page
                    copied in every layer; free_pages gives back what the forks' rows held before
  grow_pages        pages for new tokens, with the positions and slots that the append takes;
                    free_pages trims what was not accepted
"""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------- cases

def listed():
    return [
        # a short prompt of a Llama-shaped layer: latency
        dict(name="prompt_short", op="prompt", b=1, lo=40, hi=40, hq=32, hkv=8, hd=128, dtype="bf16", causal=True,
             left=-1, shape=1),
        # prompts of a serving batch, one token to some thousand, packed
        dict(name="prompt_batch", op="prompt", b=24, lo=1, hi=2100, hq=32, hkv=8, hd=128, dtype="bf16", causal=True,
             left=-1, shape=2),
        # one long document
        dict(name="prompt_long", op="prompt", b=1, lo=16384, hi=16384, hq=32, hkv=8, hd=128, dtype="bf16",
             causal=True, left=-1, shape=3),
        # a sliding layer with six heads a group and heads of 64, odd lengths
        dict(name="prompt_window", op="prompt", b=5, lo=900, hi=5003, hq=24, hkv=4, hd=64, dtype="fp16", causal=True,
             left=1023, shape=4),
        # a training step's few short sequences: latency
        dict(name="grad_short", op="grad", b=2, lo=20, hi=70, hq=32, hkv=8, hd=128, dtype="bf16", causal=True,
             left=-1, shape=5),
        # a packed training batch
        dict(name="grad_batch", op="grad", b=13, lo=30, hi=1300, hq=32, hkv=8, hd=128, dtype="bf16", causal=True,
             left=-1, shape=6),
        # one long sequence
        dict(name="grad_long", op="grad", b=1, lo=8192, hi=8192, hq=32, hkv=8, hd=128, dtype="bf16", causal=True,
             left=-1, shape=7),
        # a sliding layer, heads of 64 and a group of seven, odd lengths
        dict(name="grad_window", op="grad", b=3, lo=700, hi=2777, hq=14, hkv=2, hd=64, dtype="fp16", causal=True,
             left=511, shape=8),
        # one sequence forked into four samples, a few layers
        dict(name="fork_samples", op="fork", parents=1, children=4, hi=500, layers=4, hkv=8, hd=128, bs=16,
             pool=256, dtype="bf16", shape=9),
        # a beam of many sequences in all layers of a model
        dict(name="fork_beam", op="fork", parents=40, children=160, hi=900, layers=24, hkv=8, hd=128, bs=32,
             pool=2500, dtype="bf16", shape=10),
        # one sequence's drafted block of tokens, none accepted
        dict(name="step_one", op="step", b=1, add_lo=5, add_hi=5, hi=900, bs=16, pool=512, shape=11),
        # prompts and drafted blocks of a large batch in a large cache
        dict(name="step_batch", op="step", b=250, add_lo=1, add_hi=160, hi=4000, bs=16, pool=65536, shape=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "grad", "grad", "fork", "step"])
    if op in ("prompt", "grad"):
        hq, hkv = rng.choice([(32, 8), (16, 2), (28, 4), (8, 1), (16, 16), (40, 8), (5, 5), (6, 2)])
        hd = rng.choice([64, 64, 128, 128, 128, 80, 96, 192, 256])
        # no more products than the listed long sequences: b * hi^2 * hq * hd of theirs
        causal = rng.random() < 0.85
        most = (16384 if op == "prompt" else 8192) ** 2 * 32 * 128 // (1 if causal else 2)
        # heads of other sizes than 64 and 128 up to some thousand tokens
        top = 16384 if hd in (64, 128) else 4096
        hi = min(_log(rng, 1, top), int(math.sqrt(most / (hq * hd))))
        # nor more rows than theirs and the batches' hold, in bytes
        room = (24000 if op == "prompt" else 8192) * 128 * 40 // (hd * (hq + hkv))
        hi = min(hi, room)
        b = min(_log(rng, 1, 64), max(1, most // (hi * hi * hq * hd)), room // hi)
        left = rng.choice([-1, -1, -1, rng.randint(0, 200), _log(rng, 100, 5000)]) if causal else -1
        return dict(op=op, b=b, lo=rng.choice([hi, rng.randint(0, hi), min(hi, 1)]), hi=hi, hq=hq, hkv=hkv, hd=hd,
                    dtype=rng.choice(["bf16", "bf16", "fp16"]), causal=causal, left=left,
                    shape=rng.randint(20, 10 ** 6))
    if op == "fork":
        bs, hi, parents = rng.choice([16, 32, 48, 64]), _log(rng, 10, 900), _log(rng, 1, 40)
        hkv, hd = rng.choice([(8, 128), (2, 64), (1, 128), (4, 256), (8, 80)])
        children = _log(rng, 1, 160)
        pool = parents * (hi // bs + 1) + 2 * children + rng.randint(1, 300)
        layers = _log(rng, 1, 24)
        # no more cached bytes than in the listed beam, so no more copied ones either
        layers = max(1, min(layers, int(2500 * 32 * 8 * 128 * 24 / (pool * bs * hkv * hd))))
        children = max(1, min(children, int(160 * 32 * 8 * 128 * 24 / (bs * hkv * hd * layers))))
        return dict(op=op, parents=parents, children=children, hi=hi, layers=layers, hkv=hkv, hd=hd, bs=bs, pool=pool,
                    dtype=rng.choice(["bf16", "fp16"]), shape=rng.randint(20, 10 ** 6))
    bs, b, hi = rng.choice([16, 32, 48, 64, 256]), _log(rng, 1, 250), _log(rng, 1, 4000)
    add_hi = _log(rng, 1, max(1, min(4000, 15000 // b)))
    pool = b * ((hi + add_hi) // bs + 2) + _log(rng, 1, 20000)
    if pool > 65536:
        hi = max(1, min(hi, (40000 // b) * bs - add_hi))
        pool = 65536
    return dict(op=op, b=b, add_lo=rng.randint(0, add_hi), add_hi=add_hi, hi=hi, bs=bs, pool=pool,
                shape=rng.randint(20, 10 ** 6))


def _lengths(case):
    """Tokens of each sequence, from the case alone."""
    rng = random.Random(case["shape"])
    lens = [rng.randint(case["lo"], case["hi"]) for _ in range(case["b"])]
    return lens if sum(lens) else [1] + lens[1:]


def _seen(case):
    """(row, key) pairs that are not masked, of one head."""
    total, left = 0, case["left"]
    for n in _lengths(case):
        if not case["causal"]:
            total += n * n
        elif left < 0 or left + 1 >= n:
            total += n * (n + 1) // 2
        else:
            total += (left + 1) * (left + 2) // 2 + (n - left - 1) * (left + 1)
    return total


def _fork_lengths(case):
    """Tokens of the parents, the children's parents, tokens that the children's rows held before."""
    rng = random.Random(case["shape"])
    bs = case["bs"]
    lens = [rng.randint(1, case["hi"]) for _ in range(case["parents"])]
    src = [rng.randrange(case["parents"]) for _ in range(case["children"])]
    return lens, src, [rng.randint(0, bs) for _ in src]


def _step_lengths(case):
    """Tokens that the rows hold, and new ones."""
    rng = random.Random(case["shape"])
    return [rng.randint(0, case["hi"]) for _ in range(case["b"])], \
        [rng.randint(case["add_lo"], case["add_hi"]) for _ in range(case["b"])]


def work(case):
    if case["op"] in ("prompt", "grad"):
        rows, hq, hkv, hd = sum(_lengths(case)), case["hq"], case["hkv"], case["hd"]
        seen = _seen(case) * hq
        if case["op"] == "prompt":
            return {"bytes": 2 * rows * hd * (2 * hq + 2 * hkv) + 4 * rows * hq, "flops": 4 * hd * seen}
        return {"bytes": 2 * rows * hd * (4 * hq + 4 * hkv) + 4 * rows * hq, "flops": 10 * hd * seen}
    bs = case["bs"]
    if case["op"] == "fork":
        lens, src, before = _fork_lengths(case)
        copied = sum(lens[s] % bs for s in src) * case["layers"] * case["hkv"] * 2 * case["hd"] * 2
        entries = sum(-(-lens[s] // bs) for s in src)
        freed = sum(-(-n // bs) for n in before)
        return {"bytes": 2 * copied + 16 * entries + 12 * freed, "flops": entries + freed}
    lens, add = _step_lengths(case)
    pages = sum(-(-(n + a) // bs) - -(-n // bs) for n, a in zip(lens, add))
    return {"bytes": 16 * sum(add) + 20 * len(lens) + 20 * pages, "flops": 2 * sum(add) + pages}


# ---------------------------------------------------------------- inputs

def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if case["op"] == "fork":
        return _prepare_fork(case, gen)
    if case["op"] == "step":
        return _prepare_step(case, gen)
    dt = DTYPES[case["dtype"]]
    lens = _lengths(case)
    hq, hkv, hd, n = case["hq"], case["hkv"], case["hd"], sum(lens)
    starts = [0]
    for x in lens:
        starts.append(starts[-1] + x)
    # queries, keys and values as one projection's output holds them; channels differ in size, as keys' do
    qkv = torch.randn((n, hq + 2 * hkv, hd), generator=gen, device=DEV)
    qkv[:, hq:hq + hkv] *= torch.exp(0.4 * torch.randn(hd, generator=gen, device=DEV))
    qkv = qkv.to(dt)
    st = {"case": case, "lens": lens, "starts": starts, "scale": 1.0 / math.sqrt(hd),
          "q": qkv[:, :hq], "k": qkv[:, hq:hq + hkv], "v": qkv[:, hq + hkv:],
          "qsl": torch.tensor(starts, dtype=torch.int32, device=DEV), "window": (case["left"], -1)}
    if case["op"] == "grad":  # what the forward pass left, and the gradient that comes back
        st["dout"] = torch.randn((n, hq, hd), generator=gen, device=DEV).to(dt)
        st["out"], st["lse"] = _attend(st)
    return st


def _caches(case, gen):
    return [torch.randn((case["pool"], case["hkv"], case["bs"], 2 * case["hd"]), generator=gen, device=DEV,
                        dtype=torch.float32).to(DTYPES[case["dtype"]]) for _ in range(case["layers"])]


def _tables(lens, width, bs, pool, gen):
    """Page counts, tables and lengths of sequences that hold random pages, each its own."""
    perm = torch.randperm(pool, generator=gen, device=DEV).to(torch.int32)
    tables = torch.zeros((len(lens), width), dtype=torch.int32, device=DEV)
    refs = torch.zeros(pool, dtype=torch.int32, device=DEV)
    at = 0
    for r, x in enumerate(lens):
        m = -(-x // bs)
        tables[r, :m] = perm[at:at + m]
        at += m
    refs[perm[:at].long()] = 1
    return refs, tables, torch.tensor(lens, dtype=torch.int32, device=DEV)


def _prepare_fork(case, gen):
    lens, src, before = _fork_lengths(case)
    width = -(-case["hi"] // case["bs"]) + 2
    refs, tables, held = _tables(lens + before, width, case["bs"], case["pool"], gen)
    p = case["parents"]
    return {"case": case, "refs": refs, "tables": tables, "lens": held, "caches": _caches(case, gen),
            "src": torch.tensor(src, dtype=torch.int32, device=DEV),
            "dst": torch.arange(p, p + len(src), dtype=torch.int32, device=DEV)}


def _prepare_step(case, gen):
    lens, add = _step_lengths(case)
    width = -(-(case["hi"] + case["add_hi"]) // case["bs"]) + 1
    refs, tables, held = _tables(lens, width, case["bs"], case["pool"], gen)
    starts = [0]
    for a in add:
        starts.append(starts[-1] + a)
    return {"case": case, "refs": refs, "tables": tables, "lens": held, "keep": held.clone(), "n": starts[-1],
            "qsl": torch.tensor(starts, dtype=torch.int32, device=DEV)}


# ---------------------------------------------------------------- one pass

def run(st):
    case = st["case"]
    op = case["op"]
    if own:
        from fold_b200 import kernels
        if op == "prompt":
            out = torch.empty_like(st["q"], memory_format=torch.contiguous_format)
            lse = torch.empty((out.shape[1], out.shape[0]), device=out.device, dtype=torch.float32)
            kernels.prompt_read(st["q"], st["k"], st["v"], st["qsl"], out, softmax_scale=st["scale"],
                                causal=case["causal"], window_size=st["window"], lse=lse)
            return [out, lse]
        if op == "grad":
            return list(kernels.prompt_read_grad(st["dout"], st["q"], st["k"], st["v"], st["out"], st["lse"],
                                                 st["qsl"], softmax_scale=st["scale"], causal=case["causal"],
                                                 window_size=st["window"]))
        if op == "fork":
            kernels.free_pages(st["refs"], st["tables"], st["lens"], st["dst"], block_size=case["bs"])
            kernels.fork_pages(st["refs"], st["tables"], st["lens"], st["src"], st["dst"], st["caches"])
            return [st["refs"], st["tables"], st["lens"], *st["caches"]]
        positions, slots = kernels.grow_pages(st["refs"], st["tables"], st["lens"], st["qsl"], st["n"],
                                              block_size=case["bs"])
        kernels.free_pages(st["refs"], st["tables"], st["lens"], block_size=case["bs"], keep=st["keep"])
        return [positions, slots, st["refs"], st["tables"], st["lens"]]
    if op == "prompt":
        return list(_attend(st))
    if op == "grad":
        return _gradients(st)
    if op == "fork":
        _release(st, st["dst"].long(), torch.zeros_like(st["dst"]))
        _fork(st)
        return [st["refs"], st["tables"], st["lens"], *st["caches"]]
    positions, slots = _grow(st)
    _release(st, torch.arange(case["b"], device=DEV), st["keep"])
    return [positions, slots, st["refs"], st["tables"], st["lens"]]


def _rows_at_once(hq, n):
    return max(1, (1 << 28) // (hq * max(1, n)))  # rows whose scores fit in about a gigabyte


def _scores(st, i, a, m):
    """First key and scaled, masked scores [Hkv, m, g, keys] of rows [a, a + m) of sequence i."""
    case = st["case"]
    s0, n = st["starts"][i], st["lens"][i]
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    first = max(0, a - case["left"]) if case["left"] >= 0 else 0
    last = a + m if case["causal"] else n
    q = st["q"][s0 + a:s0 + a + m].float().reshape(m, hkv, hq // hkv, hd).permute(1, 0, 2, 3).reshape(hkv, -1, hd)
    k = st["k"][s0 + first:s0 + last].float().transpose(0, 1)
    s = (torch.matmul(q, k.transpose(1, 2)) * st["scale"]).reshape(hkv, m, hq // hkv, last - first)
    row = torch.arange(a, a + m, device=q.device)[:, None]
    key = torch.arange(first, last, device=q.device)[None, :]
    hidden = torch.zeros((m, last - first), dtype=torch.bool, device=q.device)
    if case["causal"]:
        hidden = hidden | (key > row)
    if case["left"] >= 0:
        hidden = hidden | (key < row - case["left"])
    return first, last, q, k, s.masked_fill(hidden[None, :, None, :], -math.inf)


def _attend(st):
    case = st["case"]
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    n = st["q"].shape[0]
    out = torch.zeros((n, hq, hd), device=DEV, dtype=st["q"].dtype)
    lse = torch.zeros((hq, n), device=DEV, dtype=torch.float32)
    for i, x in enumerate(st["lens"]):
        s0, step = st["starts"][i], _rows_at_once(hq, x)
        for a in range(0, x, step):
            m = min(step, x - a)
            first, last, _, _, s = _scores(st, i, a, m)
            top = s.amax(-1, keepdim=True)
            e = torch.exp(s - top)
            total = e.sum(-1, keepdim=True)
            v = st["v"][s0 + first:s0 + last].float().transpose(0, 1)
            o = torch.matmul((e / total).reshape(hkv, -1, last - first), v).reshape(hkv, m, hq // hkv, hd)
            out[s0 + a:s0 + a + m] = o.permute(1, 0, 2, 3).reshape(m, hq, hd).to(out.dtype)
            z = (top + torch.log(total))[..., 0]
            lse[:, s0 + a:s0 + a + m] = z.permute(0, 2, 1).reshape(hq, m)
    return out, lse


def _gradients(st):
    case = st["case"]
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    g, n = hq // hkv, st["q"].shape[0]
    dq = torch.zeros((n, hq, hd), device=DEV, dtype=torch.float32)
    dk = torch.zeros((n, hkv, hd), device=DEV, dtype=torch.float32)
    dv = torch.zeros((n, hkv, hd), device=DEV, dtype=torch.float32)
    for i, x in enumerate(st["lens"]):
        s0, step = st["starts"][i], _rows_at_once(hq, x) // 2 + 1
        for a in range(0, x, step):
            m = min(step, x - a)
            r = slice(s0 + a, s0 + a + m)
            first, last, q, k, s = _scores(st, i, a, m)
            top = s.amax(-1, keepdim=True)
            e = torch.exp(s - top)
            p = (e / e.sum(-1, keepdim=True)).reshape(hkv, m * g, last - first)
            v = st["v"][s0 + first:s0 + last].float().transpose(0, 1)
            do = st["dout"][r].float().reshape(m, hkv, g, hd).permute(1, 0, 2, 3).reshape(hkv, -1, hd)
            dv[s0 + first:s0 + last] += torch.matmul(p.transpose(1, 2), do).transpose(0, 1)
            dp = torch.matmul(do, v.transpose(1, 2))
            ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * st["scale"]
            dq[r] = torch.matmul(ds, k).reshape(hkv, m, g, hd).permute(1, 0, 2, 3).reshape(m, hq, hd)
            dk[s0 + first:s0 + last] += torch.matmul(ds.transpose(1, 2), q).transpose(0, 1)
    dt = st["q"].dtype
    return [dq.to(dt), dk.to(dt), dv.to(dt)]


def _pages_of(lens, bs):
    return (lens + bs - 1) // bs


def _free_order(refs):
    """Free pages, the lowest first (held ones behind them)."""
    return torch.sort((refs > 0).to(torch.int32), stable=True).indices


def _release(st, rows, keep):
    bs, lens, tables = st["case"]["bs"], st["lens"], st["tables"]
    old = lens[rows].long()
    new = torch.minimum(old, keep.long())
    j = torch.arange(tables.shape[1], device=DEV)[None]
    gone = (j >= _pages_of(new, bs)[:, None]) & (j < _pages_of(old, bs)[:, None])
    st["refs"].index_add_(0, tables[rows].long().clamp(0, st["refs"].numel() - 1).reshape(-1),
                          -gone.to(torch.int32).reshape(-1))
    lens[rows] = new.to(torch.int32)


def _take(st, rows, old_pages, new_pages):
    """Tables of the rows with their new pages, the lowest free ones in the rows' order."""
    refs = st["refs"]
    need = new_pages - old_pages
    j = torch.arange(st["tables"].shape[1], device=DEV)[None]
    fresh = (j >= old_pages[:, None]) & (j < new_pages[:, None])
    at = (torch.cumsum(need, 0) - need)[:, None] + j - old_pages[:, None]
    ids = _free_order(refs)[at.clamp(0, refs.numel() - 1)]
    refs.index_add_(0, ids.reshape(-1), fresh.to(torch.int32).reshape(-1))
    return torch.where(fresh, ids.to(torch.int32), st["tables"][rows])


def _fork(st):
    bs, lens, tables = st["case"]["bs"], st["lens"], st["tables"]
    src, dst = st["src"].long(), st["dst"].long()
    n = lens[src].long()
    full, pages = n // bs, _pages_of(n, bs)
    j = torch.arange(tables.shape[1], device=DEV)[None]
    theirs = tables[src]
    own_last = torch.gather(_take(st, dst, full, pages), 1, full[:, None])[:, 0].long()
    last = torch.gather(theirs, 1, full[:, None])[:, 0].long()
    shared = j < full[:, None]
    st["refs"].index_add_(0, theirs.long().reshape(-1), shared.to(torch.int32).reshape(-1))
    partly = pages > full
    first = theirs[:, 0].long()  # nothing to copy: a page of the parent onto itself
    to = torch.where(partly, own_last, first)
    filled = (torch.arange(bs, device=DEV)[None] < (n % bs)[:, None])[:, None, :, None]
    for c in st["caches"]:
        c[to] = torch.where(filled, c[torch.where(partly, last, first)], c[to])
    fresh = (j == full[:, None]) & partly[:, None]
    mine = torch.where(shared, theirs, tables[dst])
    tables[dst] = torch.where(fresh, own_last.to(torch.int32)[:, None], mine)
    lens[dst] = n.to(torch.int32)


def _grow(st):
    bs, lens, tables, b = st["case"]["bs"], st["lens"], st["tables"], st["case"]["b"]
    old = lens.long()
    add = (st["qsl"][1:] - st["qsl"][:-1]).long()
    rows = torch.arange(b, device=DEV)
    tables.copy_(_take(st, rows, _pages_of(old, bs), _pages_of(old + add, bs)))
    lens += add.to(torch.int32)
    t = torch.arange(st["n"], device=DEV)
    seq = torch.searchsorted(st["qsl"][1:].long().contiguous(), t, right=True)
    pos = old[seq] + t - st["qsl"].long()[seq]
    return pos, tables[seq, pos // bs].long() * bs + pos % bs


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    if case["op"] not in ("prompt", "grad"):
        return None  # page numbers and copies
    st = prepare(case, seed)
    hq, hkv, hd, left = case["hq"], case["hkv"], case["hd"], case["left"]
    g, n = hq // hkv, st["q"].shape[0]
    q, k, v = (st[x].to(torch.float64).transpose(0, 1) for x in ("q", "k", "v"))  # [heads, n, hd]
    out = torch.zeros((hq, n, hd), dtype=torch.float64, device=DEV)
    lse = torch.zeros((hq, n), dtype=torch.float64, device=DEV)
    grad = case["op"] == "grad"
    if grad:
        do = st["dout"].to(torch.float64).transpose(0, 1)
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for i, x in enumerate(st["lens"]):
        lo = st["starts"][i]
        step = max(1, (1 << 26) // max(1, x))
        for a in range(0, x, step):
            z = min(x, a + step)
            # keys that any of these rows sees
            j0 = max(0, a - left) if left >= 0 else 0
            j1 = z if case["causal"] else x
            away = torch.arange(a, z, device=DEV)[:, None] - torch.arange(j0, j1, device=DEV)[None]  # row - key
            keep = torch.ones_like(away, dtype=torch.bool)
            if case["causal"]:
                keep &= away >= 0
            if left >= 0:
                keep &= away <= left
            rows, keys = slice(lo + a, lo + z), slice(lo + j0, lo + j1)
            for h in range(hq):
                c = h // g
                logit = torch.where(keep, (q[h, rows] @ k[c, keys].T) * st["scale"],
                                    torch.full((), -math.inf, dtype=torch.float64, device=DEV))
                lse[h, rows] = torch.logsumexp(logit, dim=1)
                w = torch.exp(logit - lse[h, rows, None])
                o = w @ v[c, keys]
                out[h, rows] = o
                if grad:
                    back = do[h, rows] @ v[c, keys].T
                    dlogit = w * (back - (do[h, rows] * o).sum(1, keepdim=True)) * st["scale"]
                    dv[c, keys] += w.T @ do[h, rows]
                    dq[h, rows] = dlogit @ k[c, keys]
                    dk[c, keys] += dlogit.T @ q[h, rows]
    if grad:
        return [t.transpose(0, 1).contiguous() for t in (dq, dk, dv)]
    return [out.transpose(0, 1).contiguous(), lse]
