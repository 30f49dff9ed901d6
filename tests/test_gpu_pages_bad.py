"""Forks from rows whose table names pages that do not exist: the child stays empty, the others are served."""
import pytest
import torch

from fold_b200 import kernels
from fold_b200.errors import DEVERR_BLOCK_TABLE
from tests.test_gpu_pages import Pool, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layers", [1, 200])
@pytest.mark.parametrize("bad", [-1, -7, 100, 1 << 30])
@pytest.mark.parametrize("tokens", [700, 688])
def test_fork_from_a_bad_table(tokens, bad, layers):
    """Full pages of one parent's table (44 or 43 of 16 tokens) go wrong; the last page is partly filled or not."""
    p = Pool(100, 6, 50, 16)
    p.grow([tokens, 40, 0, 0, 0, 0])
    caches = [torch.randn(100, 1, 16, 8, device="cuda") for _ in range(layers)]
    refs, good = p.refs.clone(), p.tables.clone()
    entry = 37
    p.tables[0, entry] = bad
    kernels.fork_pages(p.refs, p.tables, p.lens, ints([0, 1, 0, 1]), ints([2, 3, 4, 5]), caches, err=p.err)
    assert int(p.err) == DEVERR_BLOCK_TABLE
    assert p.lens.tolist() == [tokens, 40, 0, 40, 0, 40]
    t = p.tables.tolist()
    assert t[3][:2] == t[5][:2] == good[1, :2].tolist()
    fresh = [t[3][2], t[5][2]]
    want = refs.clone()
    want[good[1, :2].long()] += 2
    want[fresh] += 1
    assert len(set(fresh)) == 2 and p.refs.tolist() == want.tolist()
    for c in caches[::50]:
        for page in fresh:
            assert torch.equal(c[page, :, :8], c[int(good[1, 2]), :, :8])
    # the rows that stayed empty can be forked to
    p.err.zero_()
    p.tables[0, entry] = good[0, entry]
    kernels.fork_pages(p.refs, p.tables, p.lens, ints([0, 0]), ints([2, 4]), caches, err=p.err)
    assert int(p.err) == 0 and p.lens.tolist() == [tokens, 40, tokens, 40, tokens, 40]
    full = tokens // 16
    assert p.tables[2, :full].tolist() == p.tables[4, :full].tolist() == good[0, :full].tolist()


def test_bad_partly_filled_page():
    p = Pool(8, 3, 4, 16)
    p.grow([40, 0, 0])
    refs = p.refs.tolist()
    p.tables[0, 2] = 8
    kernels.fork_pages(p.refs, p.tables, p.lens, ints([0]), ints([1]), [torch.zeros(8, 1, 16, 8, device="cuda")], err=p.err)
    assert int(p.err) == DEVERR_BLOCK_TABLE and p.lens.tolist() == [40, 0, 0] and p.refs.tolist() == refs
