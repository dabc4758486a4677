"""hq_pages_* (host memory only) with many sequences: what a call takes does not grow with the copies that wait."""
import time

import numpy as np

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
