"""States, rows and pages that lie beyond 4 GB from the start of their memory."""
import numpy as np
import pytest

from delta_ref import append, delta
from test_gpu_delta import U_MIN, inputs, split

pytestmark = pytest.mark.gpu


def test_states_in_far_slots(hqlib):
    """States of 2 MB: single tokens, chunks and parts from and to slots around 4 and 8 GB, the convolution's inputs likewise."""
    hk, hv, dk, dv, taps, slots = 1, 32, 128, 128, 8, 4100
    size, ch = hv * dk * dv * 4, 2 * hk * dk + hv * dv
    print(f"[gpu] delta slots of {slots * size >> 20} MB", flush=True)
    rng = np.random.default_rng(1)
    n_new, src, dst = [1, 70, 2100], [4099, 2048, 4098], [2047, 4097, 4096]
    T = sum(n_new)
    x, g, beta = inputs(rng, T, hk, hv, dk, dv)
    s = hqlib.DevBuf(slots * size)
    before = rng.normal(0, 0.5, (3, hv, dk, dv)).astype(np.float32)
    for i, b in zip(src, before):
        s.upload(b, offset=i * size)
    d = [hqlib.DevBuf.from_array(a) for a in (x, g, beta)]
    out = hqlib.DevBuf(T * hv * dv * 2)
    st, scan = hqlib.States(hk, hv, dk, dv, taps, slots, s, None), hqlib.Scan(3, T)
    scan.set(st, n_new, src, dst)
    hqlib.delta(scan, st, d[0], d[0].ptr + 2 * hk * dk, d[0].ptr + 4 * hk * dk, d[1], d[2], out, dk ** -0.5, qk_stride=x.shape[1], v_stride=x.shape[1])
    hqlib.synchronize()
    y = out.download((T, hv, dv), np.float16).astype(np.float64)
    q, k, v = split(x, hk, hv, dk, dv)
    for h in (0, 31):
        one = slice(h, h + 1)
        want, bound, after, e = delta(q, k, v[:, one], g[:, one], beta[:, one], [b[one] for b in before], n_new, dk ** -0.5)
        assert (np.abs(y[:, one] - want) <= bound).all()
        for i, a, b in zip(dst, after, e):
            got = s.download((1, dk, dv), np.float32, offset=i * size + h * dk * dv * 4)
            assert (np.abs(got - a) <= b + U_MIN).all(), i
    for i, b in zip(src, before):
        assert np.array_equal(s.download((hv, dk, dv), np.float32, offset=i * size), b)
    scan.free()


def test_inputs_in_far_slots(hqlib):
    """The convolution's inputs in slots around 4 GB, rows of x and of the outputs on both sides of it."""
    hk, hv, dk, dv, taps, slots = 16, 32, 128, 128, 8, 25000
    ch = 2 * hk * dk + hv * dv
    size = (taps - 1) * ch * 4
    print(f"[gpu] delta_append slots of {slots * size >> 20} MB", flush=True)
    rng = np.random.default_rng(2)
    n_new, src, dst = [5, 1, 9], [24999, 18724, -1], [18725, 24998, 24997]
    T, stride = sum(n_new), 1 << 28  # (of x: 512 MB)
    conv, x = hqlib.DevBuf(slots * size), hqlib.DevBuf(T * stride * 2)
    old = [rng.normal(0, 1, (taps - 1, ch)).astype(np.float32) for _ in range(2)]
    for i, o in zip(src, old):
        conv.upload(o, offset=i * size)
    rows = rng.normal(0, 1, (T, ch)).astype(np.float16)
    for t in range(T):
        x.upload(rows[t], offset=t * stride * 2)
    w, ab = rng.normal(0, 0.5, (ch, taps)).astype(np.float32), rng.normal(0, 1, (2, T, hv)).astype(np.float16)
    d = [hqlib.DevBuf.from_array(a) for a in (w, ab, np.zeros(hv, np.float32))]
    out, g, beta = hqlib.DevBuf(T * ch * 2), hqlib.DevBuf(T * hv * 4), hqlib.DevBuf(T * hv * 4)
    st, scan = hqlib.States(hk, hv, dk, dv, taps, slots, None, conv), hqlib.Scan(3, T)
    scan.set(st, n_new, src, dst)
    hqlib.delta_append(scan, st, x, d[0], d[1], d[1].ptr + T * hv * 2, d[2], d[2], out, g, beta, f32=False, x_stride=stride, eps=1e-6)
    hqlib.synchronize()
    zeros = np.zeros(hv, np.float32)
    want = append(rows, [*old, np.zeros((taps - 1, ch), np.float32)], w, ab[0], ab[1], zeros, zeros, n_new, hk, hv, dk, dv, 1e-6)
    assert (np.abs(out.download((T, ch), np.float16).astype(np.float64) - want[0]) <= want[1]).all()
    for i, keep in zip(dst, want[6]):
        assert np.array_equal(conv.download((taps - 1, ch), np.float32, offset=i * size), keep), i
    scan.free()


def test_far_pages(hqlib):
    """Copies between pages around 4 and 8 GB, of all and of some positions."""
    heads, hd, page, pages = 4, 256, 64, 66000
    n = page * heads * hd
    print(f"[gpu] kv_copy in {pages * n * 2 >> 20} MB", flush=True)
    rng = np.random.default_rng(3)
    k, v = hqlib.DevBuf(pages * n * 2), hqlib.DevBuf(pages * n * 2)
    src, dst, part = [65999, 0, 32768, 40000], [1, 65998, 32767, 32769], [64, 10, 64, 33]
    data = rng.normal(0, 1, (2, 4, n)).astype(np.float16)
    for buf, rows in zip((k, v), data):
        for s, t, row in zip(src, dst, rows):
            buf.upload(row, offset=s * n * 2)
            buf.upload(np.full(n, 7, np.float16), offset=t * n * 2)
    hqlib.kv_copy([hqlib.KvCache(hqlib.KV_F16, pages, page, heads, hd, k, v, (n, heads * hd, hd))], src, dst, part)
    hqlib.synchronize()
    for buf, rows in zip((k, v), data):
        for s, t, m, row in zip(src, dst, part, rows):
            m *= heads * hd
            got = buf.download(n, np.float16, offset=t * n * 2)
            assert np.array_equal(got[:m], row[:m]) and (got[m:] == 7).all() and np.array_equal(buf.download(n, np.float16, offset=s * n * 2), row), t
