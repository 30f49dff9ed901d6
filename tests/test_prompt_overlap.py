"""Outputs of the prompts' calls that share memory with an input are refused, views side by side are not (no GPU)."""
import random

import pytest

from fold_b200 import _lib
from fold_b200.errors import FoldError

FAR = 1 << 40


def grad_refused(n, hq, hkv, hd, **given):
    """Whether the gradient refuses operands (byte address, token stride, head stride), the others far apart. Without a
    workspace a call that it does not refuse ends there, before anything is launched."""
    ops = {}
    for i, name in enumerate(("do", "q", "k", "v", "o", "dq", "dk", "dv")):
        heads = hkv if name in ("k", "v", "dk", "dv") else hq
        ops[name] = given.get(name, (FAR * (i + 2), heads * hd, hd))
    args = [x for name in ("do", "q", "k", "v", "o") for x in ops[name]]
    outs = [x for name in ("dq", "dk", "dv") for x in ops[name]]
    with pytest.raises(FoldError, match="prompt read grad") as e:
        _lib.call("fold_prompt_read_grad", *args, 16, None, 16, 1, 1, -1, -1, 1.0, *outs, 0, None, 0, n, hq, hkv, hd, 0,
                  None, None)
    text = str(e.value)
    assert "share memory" in text or "workspace" in text, text
    return "share memory" in text


def elements(op, n, heads, hd):
    at, tok, head = op
    return {at // 2 + t * tok + h * head + c for t in range(n) for h in range(heads) for c in range(hd)}


def test_views_of_one_tensor():
    n, hd, base = 5, 64, 1 << 20
    row = 12 * hd  # four query heads, two of keys, two of values, four more

    def view(h):
        return base + 2 * h * hd, row, hd

    assert not grad_refused(n, 4, 2, hd, q=view(0), k=view(4), v=view(6), dq=view(8))
    for h in range(1, 12):  # from the last query head on to past the row's end
        meets = 1 <= h < 4 or h in (4, 5, 6, 7) or h > 8
        assert grad_refused(n, 4, 2, hd, q=view(0), k=view(4), v=view(6), dq=view(h)) == meets
    # the same heads first
    first = [(base + 2 * h * n * hd, hd, n * hd) for h in (0, 4, 6, 8)]
    assert not grad_refused(n, 4, 2, hd, q=first[0], k=first[1], v=first[2], dq=first[3])
    assert grad_refused(n, 4, 2, hd, q=first[0], k=first[1], v=first[2], dq=(first[3][0] - 16, hd, n * hd))
    # an output over another, and itself an input of another shape
    assert grad_refused(n, 4, 2, hd, dq=view(0), dk=view(3), dv=view(8))
    assert grad_refused(n, 4, 2, hd, k=view(0), dq=view(0))


def test_random_views():
    rng = random.Random(1)
    seen = {True: 0, False: 0}
    for _ in range(3000):
        n, hd = rng.randint(1, 6), 8 * rng.randint(1, 3)
        hkv = rng.randint(1, 3)
        hq = hkv * rng.randint(1, 3)
        if rng.random() < 0.5:  # tokens first: one stride, heads at strides of their own
            ka, kb = hd + 8 * rng.randint(0, 3), hd + 8 * rng.randint(0, 3)
            tok = max((hq - 1) * ka, (hkv - 1) * kb) + hd + 8 * rng.randint(0, 6)
            a, b = (tok, ka), (tok, kb)
        else:
            tok = hd + 8 * rng.randint(0, 2)
            head = (n - 1) * tok + hd + 8 * rng.randint(0, 4)
            a = b = (tok, head)
        base = 1 << 20
        shift = 16 * rng.randint(-60, 60)
        dq, k = (base, *a), (base + shift, *b)
        meets = bool(elements(dq, n, hq, hd) & elements(k, n, hkv, hd))
        seen[meets] += 1
        assert grad_refused(n, hq, hkv, hd, dq=dq, k=k) == meets, (n, hq, hkv, hd, dq, k)
    assert min(seen.values()) > 500


def test_other_strides():
    """Nothing that shares memory passes; what lies apart does."""
    rng = random.Random(2)
    for _ in range(2000):
        n, hd, hq, hkv = rng.randint(1, 6), 8, 4, 2
        dq = (1 << 20, 4 * hd + 8 * rng.randint(0, 4), hd)
        k = ((1 << 20) + 16 * rng.randint(-40, 40), 8 * rng.randint(0, 6), 8 * rng.randint(0, 6))
        a, b = elements(dq, n, hq, hd), elements(k, n, hkv, hd)
        refused = grad_refused(n, hq, hkv, hd, dq=dq, k=k)
        if a & b:
            assert refused
        if max(a) < min(b) or max(b) < min(a):
            assert not refused


def test_read_refuses_views_that_overlap():
    n, hd, base = 5, 64, 1 << 20
    row = 8 * hd
    for out, head in ((1, hd), (3, hd), (5, hd), (0, 2 * hd)):  # behind a query head, over keys, over values, over q apart
        o = (base + 2 * out * hd, 2 * row, head) if head != hd else (base + 2 * out * hd, row, head)
        with pytest.raises(FoldError, match="share"):
            _lib.call("fold_prompt_read", base, row, hd, base + 8 * hd, row, hd, base + 12 * hd, row, hd, 16, 1, 1, -1, -1, 1.0,
                      *o, None, n, 4, 2, hd, 0, None, None)


def test_large_sizes_do_not_wrap():
    n, hd = 1 << 28, 128
    assert not grad_refused(n, 8, 2, hd)
    whole = n * 12 * hd * 2
    q, k, v = ((1 << 20) + 2 * h * hd for h in (0, 8, 10))
    t = 12 * hd
    assert not grad_refused(n, 8, 2, hd, q=(q, t, hd), k=(k, t, hd), v=(v, t, hd), dq=((1 << 20) + whole, t, hd))
    assert grad_refused(n, 8, 2, hd, q=(q, t, hd), k=(k, t, hd), v=(v, t, hd), dq=((1 << 20) + whole - 2 * hd, t, hd))
