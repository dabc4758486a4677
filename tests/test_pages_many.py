"""hq_pages_* (host memory only) with many sequences: what a call takes does not grow with the copies that wait. And with few pages: those that
a sequence gives back are there for it."""
import time

import numpy as np
import pytest

import hq


def branch(n, page=16):
    """n sequences that branch off one within its last page and grow there, without a step in between; seconds."""
    p = hq.Pages(2 * n + 4, page, n + 1)
    p.resize(0, 0, 20)
    t = time.process_time()
    for i in range(1, n + 1):
        p.fork(0, i, 20)
        p.resize(i, 20, 21)
    for i in range(n, 0, -2):  # half of them end again before it
        p.resize(i, 0, 0)
    t = time.process_time() - t
    src, dst, m = p.copies()
    assert len(src) == n // 2 and (src == 1).all() and (m == 4).all() and len(set(dst.tolist())) == n // 2
    assert p.count(0) == (20, 2 * n + 4 - 2 - n // 2)
    table = p.table(np.arange(1, n + 1, 2), 2)
    assert (table[:, 0] == 0).all() and set(table[:, 1].tolist()) == set(dst.tolist())
    return t


def test_many_branches_between_steps():
    """2^14 and 2^17 branches: eight times the calls take some eight times as long, not sixty-four."""
    branch(1 << 10)
    few, many = min(branch(1 << 14) for _ in range(3)), branch(1 << 17)
    assert many < 24 * few, (few, many)


@pytest.mark.parametrize("keep,copied", [(10, 1), (0, 0)])
def test_writing_again_in_a_shared_page_of_a_full_pool(keep, copied):
    """A sequence that goes back into a page which others share needs one in its place: it has one among those behind, though the pool is
    empty. What it cannot have is refused as before, and nothing is changed."""
    p = hq.Pages(3, 16, 3)
    p.resize(0, 0, 16)
    p.fork(0, 1, 16)
    p.resize(1, 16, 40)
    assert p.table([1], 3).tolist() == [[0, 1, 2]] and p.count(1) == (40, 0)
    p.resize(1, keep, 12)
    row = p.table([1], 1)[0, 0]
    src, dst, n = p.copies()
    assert row in (1, 2) and p.count(1) == (12, 1) and p.table([0], 1).tolist() == [[0]]
    assert (src.tolist(), dst.tolist(), n.tolist()) == (([0], [row], [10]) if copied else ([], [], []))
    p.resize(0, 16, 17)
    assert p.count(0) == (17, 0)
    p.fork(1, 2, 12)
    for seq in (1, 2):
        with pytest.raises(hq.HQError, match="needs 1 pages more .0 are free"):
            p.resize(seq, 3, 5)
    assert p.count(2) == (12, 0) and p.table([1, 2], 1).tolist() == [[row], [row]]


def test_pages_whose_copy_waits_are_given_back_too():
    """Going back over a page that waits for its copy returns it, and the copied page that nobody holds any more with it."""
    p = hq.Pages(4, 16, 4)
    p.resize(0, 0, 20)     # 0, 1
    p.fork(0, 1, 20)
    p.resize(1, 20, 21)    # 1 is copied to 2
    p.resize(0, 0, 0)      # (1 is read by the copy, 0 is sequence 1's)
    p.fork(1, 2, 16)
    p.resize(3, 0, 16)     # 3
    assert p.table([1, 3], 2).tolist() == [[0, 2], [3, 0]] and p.count(1) == (21, 0)
    p.resize(1, 0, 5)      # page 0 is shared: one of 1 and 2 takes its place, without a copy
    assert len(p.copies()[0]) == 0 and p.count(1) == (5, 1) and p.table([2], 1).tolist() == [[0]]
    assert p.table([1], 1)[0, 0] in (1, 2)
