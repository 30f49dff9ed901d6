"""The operators of the paged path and the sizes they are measured at.

Three operators, each in a plain form (elementary torch operations in 32 bits, angles in 64) and as
the calls a user makes of fold_b200.kernels:

  rotary        rotary positions of queries and keys: half or interleaved pairs, part of the head,
                with the attention factor of scaled frequencies; `inverse` is the gradient's rotation
  append_paged  keys rotated on their way into a paged cache, values stored beside them, the same
                tokens' queries rotated in the same call
  prefix_read   attention of a batch of sequences that share a long prefix: the prefix read once for
                all rows, each sequence's own pages for its rows alone, causal over its own tokens
"""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one drafted block of four tokens of a Llama-shaped layer deep in a 128K context: latency
        dict(name="rotary_block", op="rotary", n=4, hq=32, hk=8, hd=128, rot=128, dtype="bf16", interleaved=False,
             inverse=False, theta=500000.0, factor=1.0, max_pos=131072),
        # a prompt chunk of the same layer with YaRN's attention factor
        dict(name="rotary_prompt", op="rotary", n=8192, hq=32, hk=8, hd=128, rot=128, dtype="bf16", interleaved=False,
             inverse=False, theta=500000.0, factor=1.1386, max_pos=131072),
        # the gradient of interleaved pairs on a quarter of a wide head, an odd number of tokens
        dict(name="rotary_grad_odd", op="rotary", n=3001, hq=16, hk=2, hd=256, rot=64, dtype="fp16", interleaved=True,
             inverse=True, theta=10000.0, factor=1.0, max_pos=40000),
        # a decode step of 16 sequences: one token each, queries rotated along
        dict(name="append_decode", op="append", n=16, hq=32, hkv=8, hd=128, rot=128, bs=16, dtype="bf16",
             interleaved=False, with_q=True, theta=500000.0, factor=1.0, max_pos=131072, skip=0.0),
        # a prompt of 16K tokens with padding rows
        dict(name="append_prompt", op="append", n=16384, hq=32, hkv=8, hd=128, rot=128, bs=16, dtype="bf16",
             interleaved=False, with_q=True, theta=500000.0, factor=1.0, max_pos=131072, skip=0.03),
        # heads of 80 with rotated parts of 32, interleaved, blocks of 48, keys and values alone
        dict(name="append_odd", op="append", n=1777, hq=8, hkv=5, hd=80, rot=32, bs=48, dtype="fp16",
             interleaved=True, with_q=False, theta=10000.0, factor=1.0, max_pos=9000, skip=0.1),
        # one sequence, one token, a short system prompt: latency
        dict(name="prefix_one", op="prefix", b=1, qlo=1, qhi=1, prefix=512, olo=40, ohi=40, hq=32, hkv=8, hd=128,
             bs=16, dtype="bf16", causal=True, shape=1),
        # a decode step of 64 sequences over a shared 16K prompt
        dict(name="prefix_decode", op="prefix", b=64, qlo=1, qhi=1, prefix=16384, olo=1, ohi=1024, hq=32, hkv=8,
             hd=128, bs=16, dtype="bf16", causal=True, shape=2),
        # a decode step of 256 sequences over 32K shared tokens: bound by the matrix products
        dict(name="prefix_wide", op="prefix", b=256, qlo=1, qhi=1, prefix=32768, olo=1, ohi=256, hq=32, hkv=8, hd=128,
             bs=16, dtype="bf16", causal=True, shape=3),
        # drafted blocks of one to nine tokens being checked, six heads a group, an odd prefix
        dict(name="prefix_drafts", op="prefix", b=21, qlo=1, qhi=9, prefix=6007, olo=9, ohi=900, hq=24, hkv=4, hd=64,
             bs=48, dtype="fp16", causal=True, shape=4),
        # prompts of some hundred tokens behind a shared document, heads of 256
        dict(name="prefix_extend", op="prefix", b=6, qlo=90, qhi=700, prefix=8192, olo=700, ohi=1100, hq=16, hkv=8,
             hd=256, bs=32, dtype="bf16", causal=True, shape=5),
        # three blocks of eight drafted tokens at the 128K context: bound by the prefix's bytes
        dict(name="prefix_128k", op="prefix", b=3, qlo=8, qhi=8, prefix=131072, olo=8, ohi=300, hq=32, hkv=8, hd=128,
             bs=16, dtype="bf16", causal=True, shape=6),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "prefix", "prefix"])
    if op == "prefix":
        hq, hkv = rng.choice([(32, 8), (16, 2), (28, 4), (8, 1), (16, 16), (40, 8)])
        hd = rng.choice([64, 128, 128, 256])
        qhi = rng.choice([1, 1, rng.randint(2, 12), _log(rng, 13, 500)])
        b = _log(rng, 1, 200 if qhi == 1 else max(1, min(60, 1500 // qhi)))
        prefix = rng.choice([0, _log(rng, 1, 100), _log(rng, 100, 30000), _log(rng, 100, 30000)])
        # no more products and no more cached bytes than the largest listed cases
        prefix = min(prefix, int(1e11 / (4 * hd * hq * b * qhi)))
        room = int(4.5e8 / (4 * hd * hkv)) - prefix
        ohi = max(qhi, min(_log(rng, qhi, 2500), room // b))
        return dict(op="prefix", b=b, qlo=rng.randint(1, qhi), qhi=qhi, prefix=prefix, olo=rng.randint(0, ohi),
                    ohi=ohi, hq=hq, hkv=hkv, hd=hd, bs=rng.choice([16, 32, 48, 64, 256]),
                    dtype=rng.choice(["bf16", "bf16", "fp16"]), causal=rng.random() < 0.8,
                    shape=rng.randint(10, 10 ** 6))
    hd = rng.choice([64, 80, 96, 128, 128, 256])
    rot = rng.choice([hd, hd, hd // 2, hd // 4, 2 * rng.randint(1, hd // 2)])
    rot -= rot % 2
    case = dict(op=op, n=_log(rng, 1, 8192), hd=hd, rot=rot, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                interleaved=rng.random() < 0.4, theta=rng.choice([10000.0, 500000.0, 1000000.0]),
                factor=rng.choice([1.0, 1.0, 1.2079]), max_pos=_log(rng, 10000, 131072))
    hq, hk = rng.choice([(32, 8), (16, 2), (28, 4), (8, 1), (16, 16), (7, 1)])
    if op == "rotary":
        case.update(hq=hq, hk=rng.choice([hk, hk, 0]), inverse=rng.random() < 0.4)
    else:
        case.update(hq=hq, hkv=hk, bs=rng.choice([16, 32, 48, 64, 256]), with_q=rng.random() < 0.6,
                    skip=rng.choice([0.0, 0.0, 0.2]))
    return case


def _lengths(case):
    """Query rows and own keys of each sequence, from the case alone."""
    rng = random.Random(case["shape"])
    nq = [rng.randint(case["qlo"], case["qhi"]) for _ in range(case["b"])]
    # a sequence's own keys hold at least its query tokens, as a cache does once they are appended
    keys = [max(rng.randint(case["olo"], case["ohi"]), n) for n in nq]
    return nq, keys


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "rotary":
        el = case["n"] * (case["hq"] + case["hk"])
        return {"bytes": 2 * el * case["hd"] * es + 8 * case["n"], "flops": 3 * el * case["rot"]}
    if case["op"] == "append":
        el = case["n"] * (2 * case["hkv"] + (case["hq"] if case["with_q"] else 0))
        rotated = case["n"] * (case["hkv"] + (case["hq"] if case["with_q"] else 0))
        return {"bytes": 2 * el * case["hd"] * es + 16 * case["n"], "flops": 3 * rotated * case["rot"]}
    nq, keys = _lengths(case)
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    seen = 0
    for n, o in zip(nq, keys):
        seen += n * case["prefix"] + (sum(o - n + t + 1 for t in range(n)) if case["causal"] else n * o)
    rows = sum(nq)
    return {"bytes": 2 * rows * hq * hd * es + 4 * rows * hq + 2 * (case["prefix"] + sum(keys)) * hkv * hd * es,
            "flops": 4 * hd * hq * seen}


# ---------------------------------------------------------------- inputs

def _inv_freq(case):
    i = torch.arange(0, case["rot"], 2, dtype=torch.float64)
    return (1.0 / case["theta"] ** (i / case["rot"])).float()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    host = random.Random(seed)
    dt = DTYPES[case["dtype"]]
    hd = case["hd"]

    def randn(*shape):
        return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).to(dt)

    st = {"case": case}
    if case["op"] in ("rotary", "append"):
        n = case["n"]
        first = host.randint(0, max(0, case["max_pos"] - n - 1))
        if n > 64:  # a prompt's tokens follow one another
            pos = torch.arange(first, first + n, device=DEV) % case["max_pos"]
        else:       # a step's tokens sit anywhere
            pos = torch.tensor([host.randrange(case["max_pos"]) for _ in range(n)], device=DEV)
        st["positions"] = pos.to(torch.int64)
        st["inv_freq"] = _inv_freq(case).to(DEV)
        if own:
            from fold_b200 import rope
            st["table"] = rope.rope_table(st["inv_freq"], case["max_pos"], DEV, factor=case["factor"])
    if case["op"] == "rotary":
        # queries and keys as one projection's output holds them
        qkv = randn(case["n"], case["hq"] + case["hk"], hd)
        st["q"] = qkv[:, :case["hq"]]
        st["k"] = qkv[:, case["hq"]:] if case["hk"] else None
    elif case["op"] == "append":
        n, hkv, bs = case["n"], case["hkv"], case["bs"]
        qkv = randn(n, case["hq"] + 2 * hkv, hd)
        st["q"] = qkv[:, :case["hq"]] if case["with_q"] else None
        st["k"], st["v"] = qkv[:, case["hq"]:case["hq"] + hkv], qkv[:, case["hq"] + hkv:]
        blocks = -(-n // bs)
        pool = blocks + 8
        ids = torch.randperm(pool, generator=gen, device=DEV)[:blocks]
        i = torch.arange(n, device=DEV)
        slots = ids[i // bs] * bs + i % bs
        skipped = torch.rand(n, generator=gen, device=DEV) < case["skip"]
        st["slots"] = torch.where(skipped, torch.full_like(slots, -1), slots)
        st["kv"] = randn(pool, hkv, bs, 2 * hd)
    else:
        nq, keys = _lengths(case)
        hq, hkv, bs = case["hq"], case["hkv"], case["bs"]
        pblocks = -(-case["prefix"] // bs)
        oblocks = [-(-o // bs) for o in keys]
        pool = pblocks + sum(oblocks) + 4
        perm = torch.randperm(pool, generator=gen, device=DEV).to(torch.int32)
        table = torch.zeros((case["b"], max(1, max(oblocks))), dtype=torch.int32, device=DEV)
        at = pblocks
        for s, m in enumerate(oblocks):
            table[s, :m] = perm[at:at + m]
            at += m
        st["q"] = randn(sum(nq), hq, hd)
        kv = torch.empty((pool, hkv, bs, 2 * hd), device=DEV, dtype=dt)
        scale = torch.exp(0.4 * torch.randn(2 * hd, generator=gen, device=DEV))  # channels differ in size, as keys' do
        scale[hd:] = 1.0
        for a in range(0, pool, 512):
            m = min(512, pool - a)
            kv[a:a + m] = (torch.randn((m, hkv, bs, 2 * hd), generator=gen, device=DEV) * scale).to(dt)
        starts = [0]
        for n in nq:
            starts.append(starts[-1] + n)
        st.update(kv=kv, nq=nq, keys=keys, starts=starts, scale=1.0 / math.sqrt(hd),
                  prefix_table=perm[:pblocks].clone() if pblocks else torch.zeros(1, dtype=torch.int32, device=DEV),
                  block_tables=table, qsl=torch.tensor(starts, dtype=torch.int32, device=DEV),
                  own_lens=torch.tensor(keys, dtype=torch.int32, device=DEV),
                  prefix_len=torch.tensor([case["prefix"]], dtype=torch.int32, device=DEV))
    return st


# ---------------------------------------------------------------- one pass

def run(st):
    case = st["case"]
    if own:
        from fold_b200 import kernels
        if case["op"] == "rotary":
            q, k = kernels.rotary(st["q"], st["k"], st["positions"], st["table"], interleaved=case["interleaved"],
                                  inverse=case["inverse"])
            return [q] if k is None else [q, k]
        if case["op"] == "append":
            hd = case["hd"]
            q = kernels.append_paged(st["k"], st["v"], st["positions"], st["slots"], st["kv"][..., :hd],
                                     st["kv"][..., hd:], st["table"], interleaved=case["interleaved"], q=st["q"])
            return [st["kv"]] if q is None else [st["kv"], q]
        hd = case["hd"]
        q = st["q"]
        out = torch.empty_like(q)
        lse = torch.empty((q.shape[1], q.shape[0]), device=q.device, dtype=torch.float32)
        kernels.prefix_read(q, st["qsl"], st["own_lens"], st["prefix_len"], st["kv"][..., :hd], st["kv"][..., hd:],
                            st["prefix_table"], st["block_tables"], out, softmax_scale=st["scale"],
                            causal=case["causal"], lse=lse)
        return [out, lse]
    if case["op"] == "rotary":
        cos, sin = _angles(st)
        if case["inverse"]:
            sin = -sin
        q = _rotate(st["q"], cos, sin, case["interleaved"])
        return [q] if st["k"] is None else [q, _rotate(st["k"], cos, sin, case["interleaved"])]
    if case["op"] == "append":
        cos, sin = _angles(st)
        hd, bs = case["hd"], case["bs"]
        keep = st["slots"] >= 0
        slot = st["slots"][keep]
        rows = torch.cat([_rotate(st["k"], cos, sin, case["interleaved"]), st["v"]], dim=-1)
        st["kv"][slot // bs, :, slot % bs] = rows[keep]
        if st["q"] is None:
            return [st["kv"]]
        return [st["kv"], _rotate(st["q"], cos, sin, case["interleaved"])]
    return _attend(st)


def _angles(st):
    ang = st["positions"].double()[:, None] * st["inv_freq"].double()
    f = st["case"]["factor"]
    return (torch.cos(ang) * f).float()[:, None], (torch.sin(ang) * f).float()[:, None]


def _rotate(x, cos, sin, interleaved):
    rot = 2 * cos.shape[-1]
    y = x.float().clone()
    if interleaved:
        lo, hi = y[..., 0:rot:2].clone(), y[..., 1:rot:2].clone()
        y[..., 0:rot:2] = lo * cos - hi * sin
        y[..., 1:rot:2] = hi * cos + lo * sin
    else:
        lo, hi = y[..., :rot // 2].clone(), y[..., rot // 2:rot].clone()
        y[..., :rot // 2] = lo * cos - hi * sin
        y[..., rot // 2:rot] = hi * cos + lo * sin
    return y.to(x.dtype)


def _pages(kv, table, length, hd):
    """Keys and values [Hkv, length, hd] in 32 bits of the pages in `table`."""
    bs = kv.shape[2]
    x = kv[table[:-(-length // bs)].long()].float()  # [pages, Hkv, bs, 2 hd]
    x = x.transpose(0, 1).reshape(kv.shape[1], -1, 2 * hd)[:, :length]
    return x[..., :hd], x[..., hd:]


def _attend(st):
    case = st["case"]
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    g, rows, P = hq // hkv, st["q"].shape[0], case["prefix"]
    q = st["q"].float().reshape(rows, hkv, g, hd).permute(1, 0, 2, 3)  # [Hkv, rows, g, hd]
    top = torch.full((hkv, rows, g), -math.inf, device=q.device)
    total = torch.zeros_like(top)
    acc = torch.zeros((hkv, rows, g, hd), device=q.device)
    if P:
        k, v = _pages(st["kv"], st["prefix_table"], P, hd)
        step = max(1, (1 << 28) // (hkv * g * P))  # rows whose scores fit in about a gigabyte
        for a in range(0, rows, step):
            qa = q[:, a:a + step].reshape(hkv, -1, hd)
            s = torch.matmul(qa, k.transpose(1, 2)) * st["scale"]
            m = s.amax(-1, keepdim=True)
            e = torch.exp(s - m)
            top[:, a:a + step] = m.reshape(hkv, -1, g)
            total[:, a:a + step] = e.sum(-1).reshape(hkv, -1, g)
            acc[:, a:a + step] = torch.matmul(e, v).reshape(hkv, -1, g, hd)
    for i, (n, o) in enumerate(zip(st["nq"], st["keys"])):
        if n == 0 or o == 0:
            continue
        a = st["starts"][i]
        k, v = _pages(st["kv"], st["block_tables"][i], o, hd)
        s = torch.matmul(q[:, a:a + n].reshape(hkv, n * g, hd), k.transpose(1, 2)).reshape(hkv, n, g, o) * st["scale"]
        if case["causal"]:
            last = torch.arange(n, device=q.device) + (o - n)
            s = s.masked_fill((torch.arange(o, device=q.device)[None, :] > last[:, None])[None, :, None], -math.inf)
        m = torch.maximum(s.amax(-1), top[:, a:a + n])
        shift = torch.where(torch.isinf(m), torch.zeros_like(m), m)
        e = torch.exp(s - shift[..., None])
        w = torch.exp(top[:, a:a + n] - shift)
        acc[:, a:a + n] = acc[:, a:a + n] * w[..., None] + torch.matmul(e.reshape(hkv, n * g, o), v).reshape(
            hkv, n, g, hd)
        total[:, a:a + n] = total[:, a:a + n] * w + e.sum(-1)
        top[:, a:a + n] = m
    some = total > 0
    out = torch.where(some[..., None], acc / torch.where(some, total, torch.ones_like(total))[..., None],
                      torch.zeros_like(acc))
    lse = torch.where(some, top + torch.log(total), torch.full_like(top, -math.inf))
    out = out.permute(1, 0, 2, 3).reshape(rows, hq, hd).to(st["q"].dtype)
    return [out, lse.permute(0, 2, 1).reshape(hq, rows).contiguous()]


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    hd = case["hd"]
    if case["op"] == "prefix":
        return _exact_prefix(st)
    theta = st["positions"].to(torch.float64).reshape(-1, 1, 1) * st["inv_freq"].to(torch.float64)
    turn = torch.polar(torch.full_like(theta, case["factor"]), -theta if case.get("inverse") else theta)

    def turned(x):
        x = x.to(torch.float64)
        r = case["rot"]
        if case["interleaved"]:
            z = torch.complex(x[..., 0:r:2], x[..., 1:r:2]) * turn
            head = torch.stack([z.real, z.imag], dim=-1).flatten(-2)
        else:
            z = torch.complex(x[..., :r // 2], x[..., r // 2:r]) * turn
            head = torch.cat([z.real, z.imag], dim=-1)
        return torch.cat([head, x[..., r:]], dim=-1)

    if case["op"] == "rotary":
        return [turned(x) for x in (st["q"], st["k"]) if x is not None]
    kv = st["kv"].to(torch.float64)
    flat = kv.permute(0, 2, 1, 3).reshape(-1, case["hkv"], 2 * hd)  # slots in order
    live = torch.nonzero(st["slots"] >= 0).flatten()
    flat[st["slots"][live], :, :hd] = turned(st["k"])[live]
    flat[st["slots"][live], :, hd:] = st["v"].to(torch.float64)[live]
    kv = flat.reshape(kv.shape[0], case["bs"], case["hkv"], 2 * hd).permute(0, 2, 1, 3).contiguous()
    return [kv] if st["q"] is None else [kv, turned(st["q"])]


def _exact_prefix(st):
    case = st["case"]
    hq, hd, P, bs = case["hq"], case["hd"], case["prefix"], case["bs"]
    g = hq // case["hkv"]
    rows = st["q"].shape[0]
    out = torch.zeros((rows, hq, hd), dtype=torch.float64, device=DEV)
    lse = torch.full((hq, rows), -math.inf, dtype=torch.float64, device=DEV)
    table = st["prefix_table"].to(torch.int64)
    j = torch.arange(P, device=DEV)
    for h in range(case["hkv"]):
        plane = st["kv"][:, h]  # [blocks, bs, 2 hd]
        shared = plane[table[j // bs], j % bs].to(torch.float64)
        for i, (n, o) in enumerate(zip(st["nq"], st["keys"])):
            if n == 0:
                continue
            a = st["starts"][i]
            jo = torch.arange(o, device=DEV)
            mine = plane[st["block_tables"][i].to(torch.int64)[jo // bs], jo % bs].to(torch.float64)
            seen = torch.ones((n, P + o), dtype=torch.bool, device=DEV)
            if case["causal"]:
                seen[:, P:] = (jo[None] + n) <= (o + torch.arange(n, device=DEV)[:, None])
            for c in range(g):
                x = st["q"][a:a + n, h * g + c].to(torch.float64) * st["scale"]
                logit = torch.cat([x @ shared[:, :hd].T, x @ mine[:, :hd].T], dim=1)
                logit = torch.where(seen, logit, torch.full_like(logit, -math.inf))
                z = torch.logsumexp(logit, dim=1)
                p = torch.exp(logit - torch.where(torch.isinf(z), torch.zeros_like(z), z)[:, None])
                out[a:a + n, h * g + c] = p[:, :P] @ shared[:, hd:] + p[:, P:] @ mine[:, hd:]
                lse[h * g + c, a:a + n] = z
    return [out, lse]
