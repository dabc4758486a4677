"""hq_pages_* (host memory only): which pages sequences hold as they grow, branch, shrink and end, against a model that keeps every
position's value; hq_kv_copy's refusals (host only)."""
import numpy as np
import pytest

import hq


class Model:
    """Pages with contents: every position of a sequence holds a value of its own, written into the page that the table names; the
    copies that Pages asks for are made as if at once. A sequence must always read what it wrote or took over."""

    def __init__(self, n_pages, page, n_seqs):
        self.p, self.page, self.n_pages = hq.Pages(n_pages, page, n_seqs), page, n_pages
        self.memory = np.full((n_pages, page), -1, np.int64)
        self.want = [np.empty(0, np.int64) for _ in range(n_seqs)]
        self.next = 0

    def settle(self):
        src, dst, n = self.p.copies()
        assert len(set(dst)) == len(dst) and not set(dst) & set(src) and (n > 0).all() and (n <= self.page).all()
        new = [self.memory[s, :m].copy() for s, m in zip(src, n)]
        for d, m, x in zip(dst, n, new):
            self.memory[d, :m] = x
        return len(src)

    def row(self, s):
        n = len(self.want[s])
        ld = (n + self.page - 1) // self.page
        return self.p.table([s], ld + 2)[0]

    def write(self, s, keep):
        """The positions from `keep` on, as a step appends them."""
        row = self.row(s)
        for i in range(keep, len(self.want[s])):
            self.want[s][i] = self.next
            self.memory[row[i // self.page], i % self.page] = self.next
            self.next += 1

    def check(self):
        held = {}
        for s, w in enumerate(self.want):
            n, free = self.p.count(s)
            assert n == len(w)
            row, need = self.row(s), (n + self.page - 1) // self.page
            assert (row[need:] == 0).all() and len(set(row[:need])) == need
            for p in row[:need]:
                held.setdefault(int(p), []).append(s)
            got = self.memory[row[np.arange(n) // self.page], np.arange(n) % self.page]
            assert np.array_equal(got, w), s
        assert free == self.n_pages - len(held)
        return held


@pytest.mark.parametrize("seed", range(6))
def test_any_order_of_calls(seed):
    rng = np.random.default_rng(seed)
    n_seqs, page = 7, 16
    m = Model([24, 60][seed % 2], page, n_seqs)
    refused = 0
    for _ in range(400):
        s, what = int(rng.integers(n_seqs)), rng.random()
        n = len(m.want[s])
        try:
            todo = []
            if what < 0.45:  # a few sequences grow or go back before the copies are made, as a step's sequences do
                for s in rng.permutation(n_seqs)[:rng.integers(1, 4)]:
                    n = len(m.want[s])
                    keep = n if rng.random() < 0.7 else int(rng.integers(0, n + 1))
                    new = keep + int(rng.integers(0, 50))
                    m.p.resize(int(s), keep, new)
                    m.want[s] = np.concatenate([m.want[s][:keep], np.full(new - keep, -2)])
                    todo.append((int(s), keep))
            elif what < 0.7:
                c = int(rng.integers(n_seqs))
                if len(m.want[c]) == 0 and c != s:
                    k = int(rng.integers(0, n + 1))
                    m.p.fork(s, c, k)
                    m.want[c] = m.want[s][:k].copy()
            elif what < 0.85:
                m.p.resize(s, 0, 0)
                m.want[s] = np.empty(0, np.int64)
            else:
                m.p.compact()
                m.settle()
                held = m.check()
                assert set(held) == set(range(len(held)))
        except hq.HQError as e:
            assert "pages more" in str(e)
            refused += 1
        m.settle()
        for s, keep in todo:
            m.write(s, keep)
        m.check()
    assert refused < 200
    for s in range(n_seqs):
        m.p.resize(s, 0, 0)
    m.settle()
    assert m.p.count(0) == (0, m.n_pages)


def test_copies_that_wait():
    p = hq.Pages(8, 16, 4)
    p.resize(0, 0, 20)
    assert p.table([0], 3).tolist() == [[0, 1, 0]]
    p.fork(0, 1, 20)
    p.fork(0, 2, 18)
    assert p.count(2) == (18, 6)
    # both branches grow within the shared page: two copies; the last holder keeps it as it is
    p.resize(1, 20, 21)
    p.resize(2, 18, 19)
    p.resize(0, 20, 22)
    src, dst, n = p.copies()
    assert (src.tolist(), dst.tolist(), n.tolist()) == ([1, 1], [2, 3], [4, 2])
    assert p.table([0, 1, 2], 2).tolist() == [[0, 1], [0, 2], [0, 3]]
    assert len(p.copies()[0]) == 0
    # a branch of a branch whose copy still waits reads the first page
    p.fork(1, 3, 21)
    p.resize(3, 21, 30)
    p.resize(0, 0, 0)
    p.fork(3, 0, 25)
    p.resize(0, 25, 26)
    src, dst, n = p.copies()
    assert (src.tolist(), dst.tolist(), n.tolist()) == ([2, 2], [4, 1], [5, 5])
    # a page that a waiting copy reads is not handed out before the copy has been taken
    q = hq.Pages(3, 16, 3)
    q.resize(0, 0, 10)
    q.fork(0, 1, 10)
    q.resize(1, 10, 11)
    q.resize(0, 0, 0)
    assert q.count(1) == (11, 1)
    with pytest.raises(hq.HQError, match="needs 2 pages more"):
        q.resize(2, 0, 32)
    with pytest.raises(hq.HQError, match="copies wait"):
        q.compact()
    q.copies()
    q.resize(2, 0, 32)
    assert q.table([1, 2], 2).tolist() == [[1, 0], [0, 2]]
    # a copy for a sequence that ends first is not made
    q.resize(2, 0, 0)
    q.fork(1, 2, 5)
    q.resize(2, 5, 6)
    q.resize(2, 0, 0)
    assert len(q.copies()[0]) == 0 and q.count(1) == (11, 2)
    # growing up to a page's end copies nothing; positions written again in shared pages take new ones, whole pages without a copy
    q.resize(1, 11, 16)
    q.fork(1, 2, 16)
    q.resize(2, 16, 20)
    assert len(q.copies()[0]) == 0 and q.table([2], 2).tolist() == [[1, 0]]
    q.resize(2, 0, 5)
    assert len(q.copies()[0]) == 0 and q.table([2], 1).tolist() == [[2]]


def test_refusals():
    for args, text in (((0, 16, 1), "0 pages"), ((4, 24, 1), "page_size 24"), ((4, 8, 1), "page_size 8"), ((1 << 27, 16, 1), "pages of 16"), ((4, 16, 0), "0 sequences")):
        with pytest.raises(hq.HQError, match=text):
            hq.Pages(*args)
    p = hq.Pages(4, 16, 2)
    p.resize(0, 0, 40)
    for f, text in ((lambda: p.resize(2, 0, 0), "sequence 2"), (lambda: p.resize(-1, 0, 0), "sequence -1"), (lambda: p.resize(0, 41, 50), "keep 41"), (lambda: p.resize(0, 30, 20), "keep 30"),
                    (lambda: p.resize(0, 0, 65), "have 65"), (lambda: p.resize(0, -1, 3), "keep -1"), (lambda: p.resize(1, 0, 17), "needs 2 pages more"),
                    (lambda: p.fork(0, 0, 3), "must have none"), (lambda: p.fork(1, 0, 0), "40 positions"), (lambda: p.fork(0, 1, 41), "41 positions"),
                    (lambda: p.table([0], 2), "3 pages, a row 2"), (lambda: p.table([2], 2), "sequence 2"), (lambda: p.count(5), "sequence 5")):
        with pytest.raises(hq.HQError, match=text):
            f()
    assert p.count(0) == (40, 1) and p.table([0], 3).tolist() == [[0, 1, 2]]


def test_kv_copy_refusals():
    """All of them before any device is touched."""
    def kv(n_pages=8, page=16, heads=2, hd=32, k=4096, v=8192, strides=(1024, 64, 32), type=hq.KV_F16, s=None):
        return hq.KvCache(type, n_pages, page, heads, hd, k, v, strides, s, s)
    ok = [kv()]
    for kvs, src, dst, n, text in ((ok, [0], [8], None, "page 0 to page 8"), (ok, [9], [0], None, "page 9"), (ok, [0, 1], [2, 2], None, "two copies to page 2"),
                                   (ok, [0, 2], [2, 1], None, "page 2 is read"), (ok, [3], [3], None, "page 3 is read"), (ok, [0], [1], [17], "17 positions"),
                                   (ok, [0], [1], [-1], "-1 positions"), (ok + [kv(n_pages=9)], [0], [1], None, "is not the one"), (ok + [kv(strides=(2048, 64, 32))], [0], [1], None, "differ in their strides"),
                                   ([kv(k=None)], [0], [1], None, "no memory"), ([kv(k=8)], [0], [1], None, "16-byte"), ([kv(page=24)], [0], [1], None, "page_size 24"),
                                   ([kv(strides=(1024, 60, 32))], [0], [1], None, "stride 60"), ([kv(type=hq.KV_Q8)], [0], [1], None, "scales")):
        with pytest.raises(hq.HQError, match=text):
            hq.kv_copy(kvs, src, dst, n)
    hq.kv_copy([], [0], [1])
    hq.kv_copy(ok, [], [])


def test_beam_refusals():
    """All of them before any device is touched."""
    ok = dict(logits=4096, n_groups=2, n_beams=3, V=100, score=4096, k=4, out_score=4096, out_token=4096, out_beam=4096, f32=True)
    for kw, text in ((dict(n_beams=0), "of 0 beams"), (dict(n_beams=65), "of 65 beams"), (dict(n_groups=-1), "-1 groups"), (dict(n_groups=1 << 24), "groups of 3"), (dict(V=0), "rows of 0"),
                     (dict(stride=99), "stride 99"), (dict(k=0), "k 0"), (dict(k=65), "k 65"), (dict(logits=None), "null"), (dict(score=None), "null"),
                     (dict(out_beam=None), "null"), (dict(logits=4098), "misaligned"), (dict(score=4097), "4-byte")):
        with pytest.raises(hq.HQError, match=text):
            hq.beam(**{**ok, **kw})
    hq.beam(**{**ok, "n_groups": 0})
