"""hq_kv_copy: pages and parts of pages in many caches, bit for bit, and nothing beside them."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def caches(hqlib, rng, q8, layers, pages, page, kv, hd, layout):
    """Random bits on the device and the host, with the strides of a layout."""
    row = {"pos": (page * kv * hd, kv * hd, hd), "head": (page * kv * hd, hd, page * hd), "apart": (page * (kv * hd + 16) + 32, kv * hd + 16, hd),
           "heads apart": (kv * (page * hd + 16), hd, page * hd + 16), "both apart": (page * kv * (hd + 16), kv * (hd + 16), hd + 16)}[layout]
    out = []
    for _ in range(layers):
        host = [rng.integers(0, 256 if q8 else 1 << 16, pages * row[0]).astype(np.uint8 if q8 else np.uint16) for _ in range(2)]
        scale = [rng.integers(0, 1 << 16, (pages, kv, page)).astype(np.uint16) if q8 else None for _ in range(2)]
        dev = [hqlib.DevBuf.from_array(h) for h in host] + [hqlib.DevBuf.from_array(s) if q8 else None for s in scale]
        out.append((host, scale, hqlib.KvCache(hqlib.KV_Q8 if q8 else hqlib.KV_F16, pages, page, kv, hd, dev[0], dev[1], row, dev[2], dev[3])))
    return out, row


CASES = [  # Q8, layers, pages, page size, kv heads, head_dim, layout, copies, partial
    (False, 1, 3, 16, 1, 16, "pos", 1, False), (False, 2, 40, 64, 4, 128, "pos", 15, True), (True, 3, 30, 32, 2, 96, "head", 15, True),
    (False, 17, 9, 16, 8, 64, "head", 4, True), (True, 2, 20, 128, 3, 80, "pos", 9, False), (False, 1, 12, 64, 5, 48, "apart", 6, True),
    (True, 1, 12, 64, 5, 48, "apart", 6, True), (False, 2, 12, 32, 3, 256, "heads apart", 6, True), (True, 2, 12, 32, 3, 16, "both apart", 6, True),
    (False, 1, 700, 16, 1, 32, "pos", 300, True), (True, 9, 600, 16, 1, 16, "head", 257, True), (False, 1, 4, 4096, 8, 256, "pos", 2, False),
    (False, 1, 4, 4096, 2, 64, "head", 2, True),
]


@pytest.mark.parametrize("q8,layers,pages,page,kv,hd,layout,n,partial", CASES)
def test_kv_copy(hqlib, q8, layers, pages, page, kv, hd, layout, n, partial):
    rng = np.random.default_rng(pages + n)
    cs, (ps, pos, head) = caches(hqlib, rng, q8, layers, pages, page, kv, hd, layout)
    order = rng.permutation(pages).astype(np.uint32)
    dst, src = order[:n], rng.choice(order[n:], n)  # (a source may serve several copies)
    n_pos = rng.integers(0, page + 1, n).astype(np.int32) if partial else None
    print(f"[gpu] kv_copy {layers} x {pages} pages of {page} x {kv} x {hd} {layout} q8={q8}, {n} copies", flush=True)
    hqlib.kv_copy([c[2] for c in cs], src, dst, n_pos)
    hqlib.synchronize()
    for host, scale, kvc in cs:
        for i in range(2):
            for j, (a, b) in enumerate(zip(src.tolist(), dst.tolist())):
                m = page if n_pos is None else int(n_pos[j])
                at = (np.arange(m)[:, None, None] * pos + np.arange(kv)[:, None] * head + np.arange(hd)).reshape(-1)
                host[i][b * ps + at] = host[i][a * ps + at]
                if q8:
                    scale[i][b, :, :m] = scale[i][a, :, :m]
            assert np.array_equal(kvc.keep[i].download(host[i].shape, host[i].dtype), host[i])
            if q8:
                assert np.array_equal(kvc.keep[2 + i].download(scale[i].shape, np.uint16), scale[i])


def test_on_a_stream(hqlib):
    """Copies run in the order of their stream; the lists may change when a call has returned."""
    rng = np.random.default_rng(1)
    cs, (ps, _, _) = caches(hqlib, rng, False, 1, 6, 64, 2, 64, "pos")
    s = hqlib.Stream()
    src, dst = np.array([0], np.uint32), np.array([1], np.uint32)
    for i in range(5):  # page 0 walks to page 5
        hqlib.kv_copy([cs[0][2]], src, dst, stream=s.ptr)
        src += 1
        dst += 1
    s.sync()
    got = cs[0][2].keep[0].download((6, ps), np.uint16)
    assert (got == cs[0][0][0].reshape(6, ps)[0]).all()
    s.destroy()


def test_more_caches_and_copies_than_a_launch_has(hqlib):
    test_kv_copy(hqlib, False, 45, 700, 16, 1, 16, "pos", 300, True)
