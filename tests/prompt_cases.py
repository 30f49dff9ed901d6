"""Packed prompts and their float64 oracle: attention, its gradient, and how far the kernels may be off."""
import math

import torch

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
F32 = 2.0 ** -23  # a float32 operation; tensor cores may truncate where they add
FILL = 77.0


class Prompts:
    """Sequences of the given lengths behind `lead` rows and before `rest` rows that belong to none (NaN)."""

    def __init__(self, lens, hq, hkv, hd, dtype="bf16", seed=0, lead=0, rest=0, layout="packed", boost=1.0, outlier=4.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        dt = DT[dtype]
        self.lens, self.hq, self.hkv, self.hd, self.dt, self.lead = lens, hq, hkv, hd, dt, lead
        n = lead + sum(lens) + rest
        self.n, self.u = n, torch.finfo(dt).eps / 2

        def operand(heads, size):
            x = torch.randn(n, heads, hd, generator=g, device="cuda") * size
            x[..., (seed * 7 + heads) % hd] *= outlier
            x[:lead], x[n - rest:] = math.nan, math.nan
            return x.to(dt)

        q, k, v, do = operand(hq, boost), operand(hkv, 1.0), operand(hkv, 1.0), operand(hq, 1.0)
        if layout == "packed":  # views of one projection's output
            qkv = torch.cat([q, k, v], 1)
            q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        elif layout == "heads_first":
            q, k, v, do = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v, do))
        self.q, self.k, self.v, self.do = q, k, v, do
        starts = [lead]
        for x in lens:
            starts.append(starts[-1] + x)
        self.starts = starts
        self.qsl = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.scale = hd ** -0.5

    def full(self, heads):
        return torch.full((self.n, heads, self.hd), FILL, device="cuda", dtype=self.dt)

    def outside(self):
        """Rows that belong to no sequence."""
        m = torch.ones(self.n, dtype=torch.bool, device="cuda")
        m[self.starts[0]:self.starts[-1]] = False
        return m

    def oracle(self, causal=True, window=(-1, -1), dlse=None):
        """Dict of float64 results (out, lse, dq, dk, dv) and of the bounds of the kernels' errors."""
        hq, hkv, hd, n, u, s = self.hq, self.hkv, self.hd, self.n, self.u, self.scale
        g = hq // hkv
        f64 = dict(dtype=torch.float64, device="cuda")
        r = {k: torch.full((n, hq, hd), FILL, **f64) for k in ("out", "dq")}
        r.update({k: torch.full((n, hkv, hd), FILL, **f64) for k in ("dk", "dv")}, lse=torch.full((hq, n), FILL, **f64))
        tol = {k: torch.zeros_like(x) for k, x in r.items()}
        for i, L in enumerate(self.lens):
            if L == 0:
                continue
            w = slice(self.starts[i], self.starts[i] + L)
            q, do = self.q[w].double().transpose(0, 1), self.do[w].double().transpose(0, 1)
            k, v = (x[w].double().transpose(0, 1).repeat_interleave(g, 0) for x in (self.k, self.v))
            d = torch.arange(L, device="cuda")[:, None] - torch.arange(L, device="cuda")[None]
            seen = torch.ones_like(d, dtype=torch.bool)
            left, right = window
            if causal:
                seen &= d >= 0
            if left >= 0:
                seen &= d <= left
            if right >= 0:
                seen &= -d <= right
            x = ((q * s) @ k.transpose(1, 2)).masked_fill(~seen, -math.inf)
            z = torch.logsumexp(x, 2)
            p = torch.exp(x - z[..., None])
            o, A = p @ v, p @ v.abs()
            # float32 logits: hd + 2 roundings of their terms' sizes; exponentials and running rescales a few
            # units of 2^-22 more
            mag = ((q.abs() * s) @ k.abs().transpose(1, 2)).masked_fill(~seen, 0.0)
            ex = (hd + 2) * F32 * mag.amax(2) + 2.0 ** -19
            acc = (L / 16 + 64) * F32
            # weights and result round once to the type (u each); products accumulate in float32
            to = (u + 2 * ex + acc)[..., None] * A * 1.01 + u * o.abs() + 2.0 ** -24
            r["out"][w], tol["out"][w] = o.transpose(0, 1), to.transpose(0, 1)
            r["lse"][:, w], tol["lse"][:, w] = z, 2 * ex + acc + 2.0 ** -22 * z.abs()
            # gradients; the kernels take out and lse as the forward pass left them (off by to and tl)
            tl = tol["lse"][:, w]
            delta = (do * o).sum(2)
            back = -delta if dlse is None else dlse[:, w].double() - delta
            dp = do @ v.transpose(1, 2)
            ds = p * (dp + back[..., None])
            # of a weight, relative to it: its logit, lse, the exponential
            ep = ((hd + 2) * F32 * mag + (tl + F32 * z.abs())[..., None] + 2.0 ** -19)
            e_dp = (hd + 2) * F32 * (do.abs() @ v.abs().transpose(1, 2))
            e_delta = (do.abs() * to).sum(2) + (hd + 2) * F32 * (do * o).abs().sum(2) + F32 * back.abs()
            # dS: its weight, its factor, its rounding to the type (u, or half the smallest step of fp16)
            e_ds = (ep + u) * ds.abs() * 1.01 + p * (e_dp + e_delta[..., None]) * 1.01 + seen * 2.0 ** -25
            acc_g = (g * L / 16 + 64) * F32

            def by_key(t):
                return t.reshape(hkv, g, L, hd).sum(1).transpose(0, 1)

            r["dq"][w] = (s * (ds @ k)).transpose(0, 1)
            tol["dq"][w] = (s * ((e_ds + acc * ds.abs()) @ k.abs())).transpose(0, 1)
            r["dk"][w] = by_key(s * (ds.transpose(1, 2) @ q))
            tol["dk"][w] = by_key(s * ((e_ds + acc_g * ds.abs()).transpose(1, 2) @ q.abs()))
            r["dv"][w] = by_key(p.transpose(1, 2) @ do)
            # (fp16 weights are held 2^10 up: half of the smallest step is 2^-35)
            tol["dv"][w] = by_key((p * (u + ep + acc_g) * 1.01 + seen * 2.0 ** -35).transpose(1, 2) @ do.abs())
            for name in ("dq", "dk", "dv"):  # the result's own rounding
                tol[name][w] += u * (r[name][w].abs() + tol[name][w]) + 2.0 ** -24
        return r, tol


def check(got, want, tol, what):
    got = got.double()
    assert bool(torch.isfinite(got).all()), f"{what} is not finite"
    err = (got - want).abs()
    assert bool((err <= tol).all()), f"{what} off by {float((err - tol).max())} past its tolerance"
