"""Scaled rotary frequencies and their table on the CPU, and the refusals of the rotary and paged
append entry points that need no GPU."""
import math

import numpy as np
import pytest
import torch

from fold_b200 import _lib, kernels, rope
from fold_b200.errors import FoldError

F32 = 2.0 ** -24  # half a step of float32, relative


def native(theta, d):
    return [theta ** (-2.0 * i / d) for i in range(d // 2)]


def close(got, want):
    got, want = got.numpy().astype(np.float64), np.asarray(want)
    # the float64 formulas agree to far below float32's rounding: half a step, and a little
    assert np.all(np.abs(got - want) <= 1.01 * F32 * np.abs(want))


def test_native_matches_default():
    f, c = rope.scaled_inv_freq(500000.0, 128)
    assert c == 1.0
    assert torch.equal(f, rope.default_inv_freq(500000.0, 128))


def test_linear_and_ntk():
    f, c = rope.scaled_inv_freq(10000.0, 64, {"rope_type": "linear", "factor": 4.0})
    close(f, [x / 4 for x in native(10000.0, 64)])
    assert c == 1.0
    f, c = rope.scaled_inv_freq(10000.0, 64, {"rope_type": "ntk", "factor": 8.0})
    close(f, native(10000.0 * 8.0 ** (64 / 62), 64))


def test_llama3_bands():
    L, s, a, b = 8192, 8.0, 1.0, 4.0
    f, c = rope.scaled_inv_freq(500000.0, 128, {"rope_type": "llama3", "factor": s, "low_freq_factor": a,
                                                "high_freq_factor": b, "original_max_position_embeddings": L})
    want = []
    for x in native(500000.0, 128):
        wave = 2 * math.pi / x
        if wave < L / b:
            want.append(x)
        elif wave > L / a:
            want.append(x / s)
        else:
            t = (L / wave - a) / (b - a)
            want.append((1 - t) * x / s + t * x)
    close(f, want)
    assert c == 1.0


def test_yarn_ramp_and_attention_factor():
    L, s, d, theta = 4096, 16.0, 128, 10000.0
    cfg = {"rope_type": "yarn", "factor": s, "original_max_position_embeddings": L}
    f, c = rope.scaled_inv_freq(theta, d, cfg)
    assert c == pytest.approx(0.1 * math.log(s) + 1.0, abs=1e-15)
    at = [d * math.log(L / (n * 2 * math.pi)) / (2 * math.log(theta)) for n in (32, 1)]
    lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), d - 1)
    want = []
    for i, x in enumerate(native(theta, d)):
        r = min(max((i - lo) / (hi - lo), 0.0), 1.0)
        want.append(x / s * r + x * (1 - r))
    close(f, want)
    assert f[0] == 1.0 and abs(float(f[-1]) * s / native(theta, d)[-1] - 1) < 1e-6
    assert rope.scaled_inv_freq(theta, d, {**cfg, "attention_factor": 1.25})[1] == 1.25


@pytest.mark.parametrize("theta,d,cfg", [
    (1e4, 63, None), (0.0, 64, None), (1e4, 64, {"rope_type": "magic", "factor": 2}),
    (1e4, 64, {"rope_type": "linear", "factor": 0.5}), (1e4, 2, {"rope_type": "ntk", "factor": 2}),
    (1e4, 64, {"rope_type": "llama3", "factor": 2, "low_freq_factor": 4, "high_freq_factor": 4,
               "original_max_position_embeddings": 100}),
    (1e4, 64, {"rope_type": "yarn", "factor": 2, "beta_fast": 1, "beta_slow": 1,
               "original_max_position_embeddings": 100})])
def test_scaling_refusals(theta, d, cfg):
    with pytest.raises(ValueError):
        rope.scaled_inv_freq(theta, d, cfg)


def yarn(theta, d, s, L, lo, hi):
    """YaRN's frequencies with the correction range [lo, hi] given."""
    out = []
    for i, x in enumerate(native(theta, d)):
        r = min(max((i - lo) / (hi - lo), 0.0), 1.0)
        out.append(x / s * r + x * (1 - r))
    return out


def test_yarn_correction_range_that_is_not_rounded():
    L, s, d, theta = 4096, 32.0, 64, 150000.0
    cfg = {"rope_type": "yarn", "factor": s, "original_max_position_embeddings": L, "beta_fast": 32.0,
           "beta_slow": 1.0}
    lo, hi = (d * math.log(L / (n * 2 * math.pi)) / (2 * math.log(theta)) for n in (32, 1))
    assert lo != math.floor(lo) and hi != math.ceil(hi) and 0 < lo < hi < d - 1
    close(rope.scaled_inv_freq(theta, d, {**cfg, "truncate": False})[0], yarn(theta, d, s, L, lo, hi))
    rounded = yarn(theta, d, s, L, math.floor(lo), math.ceil(hi))
    for extra in ({}, {"truncate": True}, {"truncate": None}):
        close(rope.scaled_inv_freq(theta, d, {**cfg, **extra})[0], rounded)


@pytest.mark.parametrize("s", [1.0, 4.0, 40.0])
def test_yarn_attention_factor_of_mscale(s):
    cfg = {"rope_type": "yarn", "factor": s, "original_max_position_embeddings": 4096}

    def got(**extra):
        return rope.scaled_inv_freq(10000.0, 64, {**cfg, **extra})[1]

    def scale(m):
        return 0.1 * m * math.log(s) + 1.0

    assert got(mscale=1.0, mscale_all_dim=1.0) == 1.0
    assert got(mscale=0.707, mscale_all_dim=0.707) == 1.0
    assert got(mscale=1.0, mscale_all_dim=0.5) == pytest.approx(scale(1.0) / scale(0.5), abs=1e-15)
    assert got(mscale=0.707, mscale_all_dim=1.0) == pytest.approx(scale(0.707) / scale(1.0), abs=1e-15)
    assert got() == got(mscale=1.0) == got(mscale=1.0, mscale_all_dim=0) == pytest.approx(scale(1.0), abs=1e-15)
    assert got(mscale=1.0, mscale_all_dim=0.5, attention_factor=1.25) == 1.25
    for alone in (dict(mscale=0.707), dict(mscale_all_dim=0.5), dict(mscale=0.707, mscale_all_dim=0.0)):
        with pytest.raises(ValueError, match="together"):
            got(**alone)


def test_default_is_native():
    want = rope.scaled_inv_freq(10000.0, 64)
    for cfg in ({"rope_type": "default"}, {"type": "default"}, {"rope_type": None, "type": "default"},
                {"rope_type": "default", "rope_theta": 10000, "partial_rotary_factor": 0.5, "factor": None}):
        f, c = rope.scaled_inv_freq(10000.0, 64, cfg)
        assert torch.equal(f, want[0]) and c == 1.0


@pytest.mark.parametrize("cfg,word", [
    ({"rope_type": "linear"}, "factor"), ({"rope_type": "linear", "factor": float("inf")}, "factor"),
    ({"rope_type": "default", "factor": 4.0}, "factor"), ({}, "rope_type"),
    ({"rope_type": "yarn", "factor": 4.0}, "original_max_position_embeddings"),
    ({"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 0}, "original_max_position_embeddings"),
    ({"rope_type": "llama3", "factor": 4.0, "low_freq_factor": 1, "high_freq_factor": 4},
     "original_max_position_embeddings"),
    ({"rope_type": "llama3", "factor": 4.0, "original_max_position_embeddings": 8192, "high_freq_factor": 4},
     "low_freq_factor"),
    ({"rope_type": "linear", "factor": 2.0, "alpha": 3.0}, "alpha"),
    ({"rope_type": "linear", "factor": 2.0, "attention_factor": 1.1}, "attention_factor"),
    ({"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096, "attn_factor": 0.9}, "attn_factor"),
    ({"rope_type": "default", "mrope_section": [16, 24, 24]}, "mrope_section"),
    ({"rope_type": "linear", "factor": 2.0, "rope_theta": 500000.0}, "rope_theta")])
def test_keys_that_are_missing_or_not_handled_are_refused(cfg, word):
    with pytest.raises(ValueError, match=word):
        rope.scaled_inv_freq(10000.0, 64, cfg)


def test_table_carries_the_factor():
    f = rope.default_inv_freq(10000.0, 16)
    plain, scaled = rope.rope_table(f, 64, "cpu"), rope.rope_table(f, 64, "cpu", factor=1.25)
    again = rope.rope_table(f, 64, "cpu")
    assert again is plain
    ang = np.arange(64)[:, None] * f.numpy().astype(np.float64)
    want = np.concatenate([np.cos(ang), np.sin(ang)], 1)
    assert np.abs(plain.numpy()[:64] - want).max() <= F32
    assert np.abs(scaled.numpy()[:64] - 1.25 * want).max() <= 2 * F32


@pytest.mark.parametrize("first", [torch.float32, torch.float64])
def test_tables_of_float64_frequencies_and_of_their_rounding_are_apart(first):
    f = torch.tensor([1.0, 10.0 ** -0.125, 10.0 ** -0.75 + (first is torch.float64) * 0.01], dtype=torch.float64)
    both = [f.to(first), f.to(torch.float64 if first is torch.float32 else torch.float32)]
    for x in both:  # in either order
        t = rope.rope_table(x, 131073, "cpu")
        ang = 131072.0 * x.double().numpy()
        want = np.concatenate([np.cos(ang), np.sin(ang)])
        # the angle rounds in float64 (2^-53 of 1.3e5), the entry to float32
        assert np.abs(t[131072].numpy() - want).max() <= F32 + 2.0 ** -34
    assert rope.rope_table(both[0], 100, "cpu") is not rope.rope_table(both[1], 100, "cpu")


def test_table_of_a_device_without_index_follows_the_current_one(monkeypatch):
    current, moved = [0], []
    f = rope.default_inv_freq(10000.0, 8)

    def to(self, device):
        moved.append(torch.device(device))
        return self.clone()

    monkeypatch.setattr(torch.Tensor, "to", to)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(rope, "_tables", {})
    a = rope.rope_table(f, 16, "cuda")
    current[0] = 1
    b = rope.rope_table(f, 16, "cuda")
    assert moved == [torch.device("cuda:0"), torch.device("cuda:1")] and a is not b
    assert rope.rope_table(f, 16, "cuda:0") is a and rope.rope_table(f, 16, torch.device("cuda", 1)) is b
    assert rope.rope_table(f, 16, "cuda") is b


def call_rotary(**kw):
    a = dict(q=16, hq=2, k=16, hk=1, pos=16, table=16, rows=8, rot=16, n=3, hd=32, dtype=0)
    a.update(kw)
    _lib.call("fold_rotary", a["q"], 64, 32, a["q"], 64, 32, a["hq"], a["k"], 32, 32, a["k"], 32, 32, a["hk"], a["pos"],
              a["table"], a["rows"], a["rot"], a["n"], a["hd"], a["dtype"], 0, 0, None, None)


@pytest.mark.parametrize("bad", [dict(dtype=5), dict(rot=15), dict(rot=34), dict(rot=0), dict(rows=0), dict(n=-1),
                                 dict(hd=0), dict(hq=-1), dict(pos=None), dict(table=None), dict(q=None),
                                 dict(k=None), dict(hd=16384)])
def test_rotary_refusals(bad):
    with pytest.raises(FoldError, match="rotary"):
        call_rotary(**bad)


def test_rotary_of_nothing_is_a_no_op():
    call_rotary(n=0)
    call_rotary(hq=0, hk=0)


def call_append(**kw):
    a = dict(k=16, v=16, pos=16, slots=16, kc=16, vc=16, nb=2, bs=16, table=16, rows=8, rot=16, hkv=1, hd=32, dtype=0,
             q=None, hq=0, n=3)
    a.update(kw)
    _lib.call("fold_append_paged", a["k"], 32, 32, a["v"], 32, 32, a["pos"], a["slots"], a["n"], a["kc"], a["vc"],
              a["nb"], a["bs"], 512, 512, 32, a["table"], a["rows"], a["rot"], a["hkv"], a["hd"], a["dtype"], 0, a["q"],
              64, 32, a["q"], 64, 32, a["hq"], None, None)


@pytest.mark.parametrize("bad", [dict(dtype=-1), dict(rot=33), dict(hkv=0), dict(nb=0), dict(bs=0), dict(n=-2),
                                 dict(k=None), dict(v=None), dict(slots=None), dict(kc=None), dict(vc=None),
                                 dict(pos=None), dict(hq=2), dict(hq=2, q=16, table=None)])
def test_append_refusals(bad):
    with pytest.raises(FoldError, match="paged append"):
        call_append(**bad)


def append_strides(kc=64, vc=4096, nb=2, bs=16, cs=(512, 512, 32), hkv=1, hd=32, dtype=0, qo=(64, 32), hq=0):
    _lib.call("fold_append_paged", 16, 32, 32, 16, 32, 32, 16, 16, 3, kc, vc, nb, bs, *cs, 16, 8, 16, hkv, hd, dtype, 0,
              16, 64, 32, 16, *qo, hq, None, None)


@pytest.mark.parametrize("bad", [
    dict(cs=(0, 512, 32)), dict(cs=(512, 0, 32), hkv=2), dict(cs=(512, 512, 0)), dict(cs=(31, 512, 32)),
    dict(cs=(1024, 512, 16), hkv=2), dict(cs=(-16, 512, 32)), dict(vc=64), dict(vc=64 + 62), dict(vc=64 - 62),
    dict(vc=64 + 126, dtype=2), dict(hq=2, qo=(64, 0)), dict(hq=2, qo=(1, 32))])
def test_append_refuses_slots_and_rows_that_share_memory(bad):
    with pytest.raises(FoldError, match="share memory"):
        append_strides(**bad)


@pytest.mark.parametrize("which", ["q", "k"])
@pytest.mark.parametrize("strides", [(0, 32), (64, 0), (64, 31), (1, 32), (64, -8)])
def test_rotary_refuses_output_rows_that_share_memory(which, strides):
    a, b = (strides, (64, 32)) if which == "q" else ((64, 32), strides)
    with pytest.raises(FoldError, match="share memory"):
        _lib.call("fold_rotary", 16, 64, 32, 16, *a, 2, 16, 64, 32, 16, *b, 2, 16, 16, 8, 16, 3, 32, 0, 0, 0, None, None)


def test_append_of_nothing_is_a_no_op():
    call_append(n=0)


@pytest.mark.parametrize("size,stride", [
    ((200, 2, 128), (128, 1, 1)), ((5, 3, 16), (1, 1, 1)), ((7, 4, 8), (1, 7, 1)), ((4, 2, 8), (0, 0, 1)),
    ((4, 6, 32), (0, 32, 1)), ((4, 6, 32), (192, 0, 1)), ((4, 6, 32), (32, 128, 1)), ((4, 6, 32), (192, 32, 1)),
    ((1, 1, 32), (1, 1, 1)), ((3, 2, 8), (16, 1, 2)), ((6, 1, 8), (8, 1, 1)), ((1, 6, 8), (1, 1, 1))])
def test_a_new_output_has_rows_of_its_own(size, stride):
    """Whatever the strides of the input: each row of the output is contiguous and no two share memory."""
    x = torch.zeros(40000).as_strided(size, stride)
    got, xs, out, os = kernels._rotary_out("rotary", x, None)
    assert torch.equal(got, x) and xs == got.stride() and xs[2] == 1
    assert out.shape == x.shape and os == out.stride() and os[2] == 1
    places = torch.arange(out.untyped_storage().nbytes() // 4).as_strided(size, os, out.storage_offset())
    assert places.unique().numel() == places.numel()


def test_positions_that_are_missing_are_refused(monkeypatch):
    """A rotation without positions is an argument error (the check of the device is put aside)."""
    monkeypatch.setattr(kernels, "_check_devices", lambda *a: 0)
    x, kv, i = torch.zeros(2, 1, 32), torch.zeros(1, 1, 16, 64), torch.zeros(2, dtype=torch.int64)
    t = rope.rope_table(rope.default_inv_freq(1e4, 32), 8, "cpu")
    with pytest.raises(FoldError, match="positions"):
        kernels.rotary(x, None, None, t)
    with pytest.raises(FoldError, match="positions"):
        kernels.append_paged(x, x, None, i, kv[..., :32], kv[..., 32:], t)
    with pytest.raises(FoldError, match="slots"):
        kernels.append_paged(x, x, i, None, kv[..., :32], kv[..., 32:], t)


def test_wrappers_take_cuda_tensors_only():
    x = torch.zeros(2, 1, 32)
    t = rope.rope_table(rope.default_inv_freq(1e4, 32), 8, "cpu")
    with pytest.raises(FoldError, match="CUDA"):
        kernels.rotary(x, None, torch.zeros(2, dtype=torch.int64), t)
    with pytest.raises(FoldError, match="CUDA"):
        kernels.append_paged(x, x, torch.zeros(2, dtype=torch.int64), torch.zeros(2, dtype=torch.int64),
                             torch.zeros(1, 1, 16, 32), torch.zeros(1, 1, 16, 32), t)
