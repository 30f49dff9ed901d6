"""A gradient's workspace serves every call of fewer rows with its heads and head size (no GPU)."""
import pytest

from fold_b200 import _lib
from fold_b200.errors import FoldError

FAR = 1 << 40


def enough(size, n, hq, hkv, hd, dtype=0):
    """Whether a call of n rows takes a workspace of `size` bytes. Its address is off a boundary, so that the call ends
    there, before anything is launched."""
    ops = [x for i, heads in enumerate((hq, hq, hkv, hkv, hq)) for x in (FAR * (i + 2), heads * hd, hd)]
    outs = [x for i, heads in enumerate((hq, hkv, hkv)) for x in (FAR * (i + 10), heads * hd, hd)]
    try:
        _lib.call("fold_prompt_read_grad", *ops, 16, None, 16, 1, 1, -1, -1, 1.0, *outs, 0, 8, size, n, hq, hkv, hd, dtype, None,
                  None)
    except FoldError as e:
        if "16-byte aligned" in str(e) or "workspace holds" in str(e):
            return "16-byte aligned" in str(e)
        raise
    raise AssertionError("a workspace off a boundary was taken")


@pytest.mark.parametrize("hq,hkv,hd", [(32, 8, 128), (32, 1, 64), (24, 4, 80), (12, 2, 128), (28, 4, 64), (16, 16, 128),
                                       (30, 1, 96), (32, 8, 256)])
def test_fewer_rows(hq, hkv, hd):
    # where the number of parts that a group is split into changes: tiles of 128 rows x KV heads x parts = 444
    rows = {1, 2, 127, 128, 129, 8192, 20000, 60000}
    for parts in range(1, hq // hkv + 1):
        tiles = -(-444 // (hkv * parts))
        rows |= {max(1, 128 * t + d) for t in (tiles - 1, tiles) for d in (-1, 0, 1)}
    rows = sorted(rows)
    for most in rows:
        size = _lib.prompt_read_grad_workspace(most, hq, hkv, hd)
        assert all(enough(size, n, hq, hkv, hd, dtype) for n in rows if n <= most for dtype in (0, 1))
        assert not enough(size // 4 if hd > 128 else 8 * most * hq - 16, most, hq, hkv, hd)


def test_other_heads_may_take_more():
    """A workspace is made for a call's own heads and head size."""
    size = _lib.prompt_read_grad_workspace
    assert size(2048, 32, 8, 128) > size(2048, 32, 8, 256) and size(4096, 32, 8, 128) > size(4096, 32, 32, 128)
    assert not enough(size(2048, 32, 8, 256), 2048, 32, 8, 128) and not enough(size(4096, 32, 32, 128), 4096, 32, 8, 128)


def test_heads_past_the_grid():
    """Above head size 128 heads of queries and keys together are up to 65535."""
    size = _lib.prompt_read_grad_workspace
    for hq, hkv in ((40000, 40000), (65535, 1)):
        assert size(1, hq, hkv, 256) == size(1, hq, hkv, 136) == -1 and size(1, hq, hkv, 128) > 0
        with pytest.raises(FoldError, match="too many heads"):
            enough(1 << 40, 1, hq, hkv, 256)
    assert size(1, 65534, 1, 256) > 0
