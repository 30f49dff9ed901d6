"""Rotary frequencies of a drafter layer and the cos/sin table the far-query rotation reads.

drafter_rope follows fold/rope.py:14-28 of the reference (neox-style default or Gemma-4
proportional rotary modules only; scaled variants are rejected because FOLD re-rotates queries
with the native frequencies).

rope_table is the device table of the rotation: float32 [rows, rotary_dim] with cos(p f_i) in the
first half and sin(p f_i) in the second, the layout of vLLM's cos_sin_cache. It is formed in
float64 on the host, so the rotation by (D - H) stays exact to float32 at offsets of 1e5 and more
(the reference's kernel forms that angle in float32). Tables are shared by every layer with the
same frequencies on a device.
"""
from __future__ import annotations

import threading
from dataclasses import dataclass

import numpy as np
import torch


@dataclass(frozen=True)
class Rope:
    inv_freq: torch.Tensor  # [rotary_dim / 2], float32
    rotary_dim: int
    head_dim: int


def drafter_rope(rotary_emb, device=None) -> Rope:
    """Frequencies of a vLLM rotary module (RotaryEmbedding or Gemma4RotaryEmbedding, neox)."""
    name = type(rotary_emb).__name__
    if name not in {"RotaryEmbedding", "Gemma4RotaryEmbedding"}:
        raise ValueError(f"unsupported rotary embedding: {name}")
    if not rotary_emb.is_neox_style:
        raise ValueError("only neox-style rotary embeddings are supported")
    freq = rotary_emb._compute_inv_freq(float(rotary_emb.base)).detach().clone()
    freq = freq.to(device=device or rotary_emb.cos_sin_cache.device, dtype=torch.float32)
    dim = int(rotary_emb.rotary_dim)
    if dim != 2 * freq.numel() or not 0 < dim <= rotary_emb.head_size:
        raise ValueError("rotary and head dimensions disagree")
    return Rope(freq, dim, int(rotary_emb.head_size))


def default_inv_freq(theta: float, rotary_dim: int, device=None) -> torch.Tensor:
    """1 / theta^(2i / rotary_dim) as float32 (vLLM's default RotaryEmbedding)."""
    i = np.arange(0, rotary_dim, 2, dtype=np.float64)
    return torch.from_numpy((1.0 / (theta ** (i / rotary_dim))).astype(np.float32)).to(device)


# Keys of each rule, and keys that any of them may carry.
_SCALING_KEYS = {
    "default": set(),
    "linear": set(),
    "ntk": set(),
    "llama3": {"low_freq_factor", "high_freq_factor"},
    "yarn": {"beta_fast", "beta_slow", "truncate", "attention_factor", "mscale", "mscale_all_dim"},
}
_COMMON_KEYS = {"rope_type", "type", "factor", "rope_theta", "original_max_position_embeddings",
                "max_position_embeddings", "partial_rotary_factor", "finetuned"}


def _yarn_attention(given, s):
    """YaRN's attention factor for contexts s times the trained one."""
    if "attention_factor" in given:
        return float(given["attention_factor"])
    m, a = float(given.get("mscale", 0.0)), float(given.get("mscale_all_dim", 0.0))
    if m and a:
        return (0.1 * m * np.log(s) + 1.0) / (0.1 * a * np.log(s) + 1.0)
    if a or m not in (0.0, 1.0):  # mscale 1 alone is the plain factor by every definition
        raise ValueError("scaled_inv_freq: yarn takes mscale and mscale_all_dim together")
    return 0.1 * np.log(s) + 1.0


def scaled_inv_freq(theta: float, rotary_dim: int, scaling=None, device=None):
    """(frequencies float32 [rotary_dim / 2], attention factor) of a long-context rotary scaling, for
    rope_table(inv_freq, rows, device, factor). `scaling` is None (native) or a dict in the form
    model configurations give it:

      {"rope_type": "default"}                 native
      {"rope_type": "linear", "factor": s}     positions interpolated: f / s
      {"rope_type": "ntk", "factor": s}        base stretched: theta * s^(d / (d - 2))
      {"rope_type": "llama3", "factor": s, "low_freq_factor": a, "high_freq_factor": b,
       "original_max_position_embeddings": L}  f / s below a turns in L, f above b, linear between
      {"rope_type": "yarn", "factor": s, "original_max_position_embeddings": L, "beta_fast": 32,
       "beta_slow": 1}                         f above beta_fast turns in L, f / s below beta_slow,
                                               a linear ramp over the dims between, its ends at whole
                                               dims unless "truncate" is false; the attention factor is
                                               "attention_factor" where given, else 0.1 ln s + 1, or
                                               with "mscale" m and "mscale_all_dim" a
                                               (0.1 m ln s + 1) / (0.1 a ln s + 1)

    Keys that say nothing about the rotation's angles (the trained or the longest context beside a rule
    that does not use it, the part of the head that is rotated) may be there, as may a "rope_theta"
    equal to theta. Any other key, and one of mscale and mscale_all_dim alone (definitions of it
    differ), is refused, since leaving it out would give other frequencies than the model's.
    """
    d = int(rotary_dim)
    if d < 2 or d % 2 or not theta > 0:
        raise ValueError("scaled_inv_freq: rotary_dim must be even and positive, theta positive")
    i = np.arange(0, d, 2, dtype=np.float64)
    f = 1.0 / (float(theta) ** (i / d))
    attention = 1.0
    if scaling is not None:
        kind = scaling.get("rope_type") or scaling.get("type")
        if kind not in _SCALING_KEYS:
            raise ValueError(f"scaled_inv_freq: unknown rope_type {kind!r}")
        given = {k: v for k, v in scaling.items() if v is not None}
        unknown = sorted(set(given) - _COMMON_KEYS - _SCALING_KEYS[kind])
        if unknown:
            raise ValueError(f"scaled_inv_freq: {kind} does not take {', '.join(unknown)}")
        if float(given.get("rope_theta", theta)) != float(theta):
            raise ValueError(f"scaled_inv_freq: theta {theta} is not the scaling's rope_theta {given['rope_theta']}")

        def need(key):
            if key not in given:
                raise ValueError(f"scaled_inv_freq: {kind} needs {key}")
            return float(given[key])

        s = float(given.get("factor", 1.0)) if kind == "default" else need("factor")
        if not 1.0 <= s < np.inf or (kind == "default" and s != 1.0):
            raise ValueError("scaled_inv_freq: factor must be finite and at least 1, of default 1")
        if kind == "linear":
            f = f / s
        elif kind == "ntk":
            if d < 4:
                raise ValueError("scaled_inv_freq: ntk needs a rotary_dim of at least 4")
            f = 1.0 / ((float(theta) * s ** (d / (d - 2))) ** (i / d))
        elif kind != "default":
            ctx = need("original_max_position_embeddings")
            if not 0 < ctx < np.inf:
                raise ValueError("scaled_inv_freq: original_max_position_embeddings must be positive")
            turns = ctx * f / (2.0 * np.pi)  # whole turns of each pair over the trained context
            if kind == "llama3":
                lo, hi = need("low_freq_factor"), need("high_freq_factor")
                if not hi > lo > 0:
                    raise ValueError("scaled_inv_freq: llama3 needs high_freq_factor > low_freq_factor > 0")
                keep = np.clip((turns - lo) / (hi - lo), 0.0, 1.0)
            else:
                fast, slow = float(given.get("beta_fast", 32)), float(given.get("beta_slow", 1))
                if not fast > slow > 0 or not theta > 1:
                    raise ValueError("scaled_inv_freq: yarn needs beta_fast > beta_slow > 0 and theta > 1")

                def dim_of(n):  # the (real-valued) pair index that makes n turns
                    return d * np.log(ctx / (n * 2.0 * np.pi)) / (2.0 * np.log(float(theta)))

                lo, hi = dim_of(fast), dim_of(slow)
                if given.get("truncate", True):
                    lo, hi = np.floor(lo), np.ceil(hi)
                lo, hi = max(lo, 0.0), min(hi, d - 1.0)
                ramp = (np.arange(d // 2) - lo) / max(hi - lo, 1e-3)
                keep = 1.0 - np.clip(ramp, 0.0, 1.0)
                attention = _yarn_attention(given, s)
            f = f * keep + (f / s) * (1.0 - keep)
    return torch.from_numpy(f.astype(np.float32)).to(device), float(attention)


def table_host(inv_freq, rows: int, factor: float = 1.0) -> np.ndarray:
    """cos/sin table [rows, 2 * len(inv_freq)] float32 times `factor`, computed in float64."""
    f = np.asarray(inv_freq.detach().cpu() if isinstance(inv_freq, torch.Tensor) else inv_freq, dtype=np.float64)
    out = np.empty((rows, 2 * f.size), dtype=np.float32)
    step = 1 << 16
    for a in range(0, rows, step):
        ang = np.arange(a, min(rows, a + step), dtype=np.float64)[:, None] * f[None, :]
        out[a:a + ang.shape[0], :f.size] = np.cos(ang) * factor
        out[a:a + ang.shape[0], f.size:] = np.sin(ang) * factor
    return out


_tables: dict = {}
_tables_lock = threading.Lock()


def rope_table(inv_freq: torch.Tensor, rows: int, device, factor: float = 1.0) -> torch.Tensor:
    """Shared device table with at least `rows` rows for these frequencies and this attention
    factor (scaled_inv_freq). A call that asks for more rows makes a new table: a captured graph's
    owner keeps the one it was captured with."""
    device = torch.device(device)
    if device.type == "cuda" and device.index is None:  # one table a device, whichever is current
        device = torch.device("cuda", torch.cuda.current_device())
    # the frequencies as the table is computed from them: float64 ones and their float32 rounding
    # lie 4e-3 rad apart at position 131072
    key = (np.asarray(inv_freq.detach().cpu(), dtype=np.float64).tobytes(), str(device), float(factor))
    with _tables_lock:
        t = _tables.get(key)
        if t is None or t.shape[0] < rows:
            t = torch.from_numpy(table_host(inv_freq, rows, factor)).to(device)
            _tables[key] = t
        return t
