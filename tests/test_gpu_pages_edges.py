"""GPU: what the page operators do with requests that touch one another, table by table."""

from __future__ import annotations

import pytest
import torch

from rows_helpers import i32
from test_gpu_cache_pages import _bytes, _cache

pytestmark = pytest.mark.gpu


def _ops():
    from specdec_b200.kernels import ops

    return ops


def _state(c):
    return c.page_table.cpu().tolist(), c.lengths.cpu().tolist(), c.page_refs.cpu().tolist()


@pytest.mark.parametrize("order", [(0, 1), (1, 0)])
def test_chains_of_forks(order):
    """Of 0 -> 1 and 1 -> 2 the first runs, in whatever order they are listed, and 2 stays as it was."""
    from specdec_b200 import _lib

    c = _cache(4, 20, 64)
    c.reserve([40, 20, 10, 0])
    c.lengths.copy_(i32([40, 20, 10, 0]))
    first = _bytes(c)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    pairs = [((0, 1, 40), (1, 2, 20))[i] for i in order]
    c.fork(*map(list, zip(*pairs)), status=status)
    assert int(status) == _lib.STATUS_BAD_SEQUENCE
    table, lengths, refs = _state(c)
    # sequence 0: pages 0 .. 2; 1 held 3 and 4; 2 holds 5; the copy of page 2 is the lowest free page, 3
    assert table == [[0, 1, 2, -1], [0, 1, 3, -1], [5, -1, -1, -1], [-1] * 4] and lengths == [40, 40, 10, 0]
    assert refs[:6] == [2, 2, 1, 1, 0, 1]
    now = _bytes(c)
    assert torch.equal(now[3], first[2]) and torch.equal(now[[0, 1, 2, 5]], first[[0, 1, 2, 5]])


def test_rings_and_doubles_of_forks():
    from specdec_b200 import _lib

    for pairs, want in [(((0, 1, 16), (1, 0, 16)), [16, 32, 5, 0]),      # each source is the other's target
                        (((0, 0, 16),), [16, 32, 5, 0]),                 # itself
                        (((0, 3, 16), (1, 3, 32)), [16, 32, 5, 16]),     # one target twice: the first
                        (((0, 3, 99), (1, 3, 32)), [16, 32, 5, 0]),      # also where the first is left out
                        (((0, 9, 16), (9, 1, 1), (2, 3, 5)), [16, 32, 5, 5])]:  # no sequences, and one that is fine
        c = _cache(4, 20, 64)
        c.reserve([16, 32, 5, 0])
        c.lengths.copy_(i32([16, 32, 5, 0]))
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        c.fork(*map(list, zip(*pairs)), status=status)
        assert int(status) == _lib.STATUS_BAD_SEQUENCE
        table, lengths, refs = _state(c)
        assert lengths == want, pairs
        held = [p for row in table for p in row if p >= 0]
        assert [held.count(p) for p in range(20)] == refs


def test_a_page_that_all_its_holders_write_into():
    """Both go on in a page that they share: both get new ones, judged by the counts before the call, and the page is free
    after it; where only one new page is left the second is refused, and gets by in a second call."""
    from specdec_b200 import _lib

    for pages in (10, 2):
        c = _cache(2, pages, 32)
        c.reserve([16, 0])
        c.lengths.copy_(i32([16, 0]))
        c.fork([0], [1], [16])
        c.lengths.copy_(i32([8, 8]))
        first = _bytes(c)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        c.reserve([16, 16], status=status)
        table, _, refs = _state(c)
        if pages == 10:
            assert int(status) == 0 and table == [[1, -1], [2, -1]] and refs[:3] == [0, 1, 1]
            assert torch.equal(_bytes(c)[1:3], first[[0, 0]])
        else:
            assert int(status) == _lib.STATUS_NO_PAGES and table == [[1, -1], [0, -1]] and refs == [1, 1]
            status.zero_()
            c.reserve([16, 16], status=status)
            assert int(status) == 0 and _state(c)[0] == [[1, -1], [0, -1]]
