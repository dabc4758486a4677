"""hq_delta_append against float64 (tests/delta_ref.py): convolution, norms, gates and the inputs that stay in the slots."""
import numpy as np
import pytest

from delta_ref import append

pytestmark = pytest.mark.gpu

# key heads, value heads, k_dim, v_dim, taps, f32, (new tokens, slot before, slot after) of each sequence
CASES = [
    (1, 1, 16, 16, 4, True, [(1, -1, 0)]),
    (1, 2, 64, 64, 4, False, [(1, 3, 3), (2, -1, 1), (0, 4, 2), (3, 0, 0)]),
    (16, 32, 128, 128, 4, True, [(1, 0, 0), (9, 1, 5), (8, -1, 2), (0, 6, -1), (7, 3, -1), (0, -1, 4)]),
    (2, 4, 96, 192, 2, True, [(17, 1, 1), (1, -1, 0)]),
    (3, 3, 48, 80, 8, False, [(5, 0, 0), (1, 1, 2), (30, -1, 3)]),
    (1, 4, 256, 256, 3, True, [(10, 0, 1), (2, 2, 2)]),
    (2, 2, 32, 16, 1, False, [(4, -1, -1), (3, 0, 0)]),
    (4, 8, 64, 128, 5, True, [(1, 1, 1), (4, 2, 3), (3, -1, 0)]),
    (1, 1, 128, 128, 4, True, [(260, 0, 0)]),
]


@pytest.mark.parametrize("hk,hv,dk,dv,taps,f32,seqs", CASES)
def test_delta_append(hqlib, hk, hv, dk, dv, taps, f32, seqs):
    rng = np.random.default_rng(hk * dk + taps)
    n_new, src, dst = [list(a) for a in zip(*seqs)]
    T, ch, slots, eps = sum(n_new), 2 * hk * dk + hv * dv, 8, 1e-5
    dt_ = np.float32 if f32 else np.float16
    x = rng.normal(0, 1, (T + 2, ch + 8)).astype(dt_)  # rows and values of other use behind them
    ab = rng.normal(0, 3, (T + 2, 2, hv + 1)).astype(dt_)
    w = rng.normal(0, 0.5, (ch, taps)).astype(np.float32)
    a_log, dt = rng.normal(0, 1, hv).astype(np.float32), rng.normal(-2, 2, hv).astype(np.float32)
    conv = np.full((slots, taps - 1, ch), np.nan, np.float32)
    for s in src:
        if s >= 0:
            conv[s] = rng.normal(0, 1, (taps - 1, ch))
    old = [conv[s] if s >= 0 else np.zeros((taps - 1, ch), np.float32) for s in src]
    d = [hqlib.DevBuf.from_array(a) for a in (x, ab, w, a_log, dt, conv)]
    st = hqlib.States(hk, hv, dk, dv, taps, slots, None, d[5])
    scan = hqlib.Scan(len(seqs), T)
    scan.set(st, n_new, src, dst)
    fill = np.full((T + 1, ch), 7, np.float16)
    out, g, beta = hqlib.DevBuf.from_array(fill), hqlib.DevBuf.from_array(np.full((T + 1, hv), 7, np.float32)), hqlib.DevBuf.from_array(np.full((T + 1, hv), 7, np.float32))
    print(f"[gpu] delta_append {hk}/{hv} x {dk}, {dv} taps {taps} {seqs}", flush=True)
    hqlib.delta_append(scan, st, d[0], d[2], d[1], d[1].ptr + (hv + 1) * ab.itemsize, d[3], d[4], out, g, beta, f32=f32, x_stride=ch + 8,
                       ab_stride=2 * (hv + 1), eps=eps)
    hqlib.synchronize()
    want = append(x[:T, :ch], old, w, ab[:T, 0, :hv], ab[:T, 1, :hv], a_log, dt, n_new, hk, hv, dk, dv, eps)
    for buf, dtype, y, b in ((out, np.float16, want[0], want[1]), (g, np.float32, want[2], want[3]), (beta, np.float32, want[4], want[5])):
        got = buf.download((T + 1, y.shape[1]), dtype)
        assert (got[T] == 7).all()  # behind the last token
        assert (np.abs(got[:T].astype(np.float64) - y) <= b).all()
    for s, k in zip(dst, want[6]):
        if s >= 0:
            conv[s] = k
    assert np.array_equal(d[5].download(conv.shape, np.float32).view(np.uint32), conv.view(np.uint32))  # and nothing else was written
    scan.free()


def test_far_gates(hqlib):
    """Gates far from zero: the logarithm of a decay never overflows on its way, a write strength ends at 0 and 1."""
    hk = hv = 8
    st = hqlib.States(hk, hv, 16, 16, 1, 1, None, None)
    scan = hqlib.Scan(1, 1)
    scan.set(st, [1], [-1], [-1])
    a = np.array([-200, -90, -20, 0, 20, 90, 1e4, 3e38], np.float32)
    b = np.array([-3e38, -200, -90, 0, 10, 90, 200, 3e38], np.float32)
    d = [hqlib.DevBuf.from_array(x) for x in (np.ones(384, np.float32), np.ones(384, np.float32), a, b, np.zeros(8, np.float32))]
    out = [hqlib.DevBuf(n) for n in (384 * 2, 32, 32)]
    hqlib.delta_append(scan, st, d[0], d[1], d[2], d[3], d[4], d[4], *out, f32=True)
    hqlib.synchronize()
    g, beta = (o.download(8, np.float32).astype(np.float64) for o in out[1:])
    y, w = np.logaddexp(0, a.astype(np.float64)), np.exp(-np.logaddexp(0, -b.astype(np.float64)))
    assert (np.abs(g + y) <= 2.0 ** -20 * y + 2.0 ** -126).all() and (np.abs(beta - w) <= 2.0 ** -20 * w + 2.0 ** -126).all()
    scan.free()


def test_refusals(hqlib):
    S, D = hqlib.States, hqlib.DevBuf
    for args, text in (((2, 3, 64, 64, 4, 4), "3 value heads over 2"), ((1, 1, 24, 64, 4, 4), "heads of 24"), ((1, 1, 64, 272, 4, 4), "272"),
                       ((1, 1, 64, 64, 9, 4), "9 taps"), ((1, 1, 64, 64, 0, 4), "0 taps"), ((1, 1, 64, 64, 4, 0), "0 slots")):
        with pytest.raises(hqlib.HQError, match=text):
            hqlib.Scan(2, 8).set(S(*args, None, None), [1], [-1], [0])
    with pytest.raises(hqlib.HQError, match="0 sequences"):
        hqlib.Scan(0, 8)
    st = S(1, 1, 64, 64, 4, 4, None, D(4 * 3 * 192 * 4))
    scan = hqlib.Scan(3, 8)
    for args, text in ((([1] * 4, [-1] * 4, [0, 1, 2, 3]), "4 sequences"), (([9], [-1], [0]), "9 new tokens"), (([-1], [-1], [0]), "-1 new"),
                       (([1], [4], [0]), "from slot 4"), (([1], [-1], [4]), "to slot 4"), (([1], [-2], [0]), "from slot -2"),
                       (([1, 1], [-1, -1], [2, 2]), "0 and 1 leave their states in slot 2"),
                       (([1, 1], [2, 1], [2, 2]), "in slot 2"), (([1, 0], [2, 2], [3, 2]), "sequence 0 goes on from slot 2, where sequence 1")):
        with pytest.raises(hqlib.HQError, match=text):
            scan.set(st, *args)
    x = D(64 * 192 * 4)
    ok = dict(scan=scan, states=st, x=x, conv_w=x, a=x, b=x, a_log=x, dt_bias=x, qkv=x, decay=x, beta=x, f32=True)
    with pytest.raises(hqlib.HQError, match="no step"):
        hqlib.delta_append(**ok)
    scan.set(st, [1, 2], [-1, 3], [0, 1])
    for kw, text in ((dict(x=x.ptr + 8), "16-byte"), (dict(x_stride=196), "stride"), (dict(x_stride=-8), "stride"), (dict(qkv=x.ptr + 2), "16-byte"), (dict(x=None), "null"),
                     (dict(beta=None), "null"), (dict(conv_w=x.ptr + 4), "weights"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(a=x.ptr + 2), "misaligned"),
                     (dict(states=S(1, 1, 64, 64, 4, 4, None, None)), "memory of the convolution"), (dict(states=S(1, 1, 64, 64, 3, 4, None, x)), "not those"),
                     (dict(states=S(1, 1, 64, 64, 4, 5, None, x)), "not those")):
        with pytest.raises(hqlib.HQError, match=text):
            hqlib.delta_append(**{**ok, **kw})
    # a step of nothing is one
    scan.set(st, [], [], [])
    hqlib.delta_append(**ok)
    scan.set(st, [0, 0], [1, -1], [1, -1])
    hqlib.delta_append(**ok)
    hqlib.synchronize()
    scan.free()
