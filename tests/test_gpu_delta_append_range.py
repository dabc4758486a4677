"""hq_delta_append where the squares of a head's values pass fp32's range or vanish in it: queries and keys have a norm of 1 (below it where
eps counts) all the same, within delta_ref's bounds."""
import numpy as np
import pytest

from delta_ref import append

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hk,hv,dk,dv,taps", [(1, 1, 128, 128, 4), (2, 2, 16, 32, 2), (1, 2, 96, 192, 8), (1, 1, 256, 64, 4)])
@pytest.mark.parametrize("size,eps", [(1.0, 1e-6), (1e15, 1e-6), (1e19, 1e-6), (1e25, 0.0), (1e33, 1e-6), (1e-16, 0.0), (1e-22, 0.0), (1e-30, 0.0), (1e-20, 1e-38), (1e-30, 1e-6)])
def test_sizes_of_inputs(hqlib, hk, hv, dk, dv, taps, size, eps):
    rng = np.random.default_rng(dk + taps)
    n_new, T, ch = [19, 3], 22, 2 * hk * dk + hv * dv
    x = rng.normal(0, 1, (T, ch)).astype(np.float32)
    x[:, :2 * hk * dk] *= np.float32(size)
    w = np.abs(rng.normal(0, 0.5, (ch, taps))).astype(np.float32)
    x[:, :2 * hk * dk] = np.abs(x[:, :2 * hk * dk])  # (nothing cancels: a float64 sum has the sign that silu takes to 0 or to its size)
    conv = np.zeros((2, taps - 1, ch), np.float32)
    conv[1] = rng.normal(0, 1, (taps - 1, ch))
    conv[1, :, :2 * hk * dk] = np.abs(conv[1, :, :2 * hk * dk]) * np.float32(size)
    ab, a_log, dt = rng.normal(0, 1, (2, T, hv)).astype(np.float32), np.zeros(hv, np.float32), np.zeros(hv, np.float32)
    d = [hqlib.DevBuf.from_array(a) for a in (x, w, ab, a_log, dt, conv)]
    st, scan = hqlib.States(hk, hv, dk, dv, taps, 2, None, d[5]), hqlib.Scan(2, T)
    scan.set(st, n_new, [-1, 1], [-1, -1])
    out, g, beta = hqlib.DevBuf(T * ch * 2), hqlib.DevBuf(T * hv * 4), hqlib.DevBuf(T * hv * 4)
    print(f"[gpu] delta_append {hk}/{hv} x {dk}, {dv} taps {taps} inputs of {size} eps={eps}", flush=True)
    hqlib.delta_append(scan, st, d[0], d[1], d[2], d[2].ptr + T * hv * 4, d[3], d[4], out, g, beta, f32=True, eps=eps)
    hqlib.synchronize()
    want = append(x, [np.zeros((taps - 1, ch), np.float32), conv[1]], w, ab[0], ab[1], a_log, dt, n_new, hk, hv, dk, dv, float(np.float32(eps)))
    got = out.download((T, ch), np.float16).astype(np.float64)
    assert (np.abs(got - want[0]) <= want[1]).all()
    if eps == 0 or size > 1:
        assert (np.abs(np.linalg.norm(got[:, :2 * hk * dk].reshape(T, 2 * hk, dk), axis=-1) - 1) < 2.0 ** -9).all()
    scan.free()


def test_heads_of_zeros(hqlib):
    """All inputs of a head 0: zeros, for eps above 0."""
    hk, hv, dk, dv, T = 1, 1, 64, 64, 9
    ch = 2 * hk * dk + hv * dv
    x = np.ones((T, ch), np.float32)
    x[:, :dk] = 0
    d = [hqlib.DevBuf.from_array(a) for a in (x, np.ones((ch, 4), np.float32), np.zeros((T, hv), np.float32), np.zeros(hv, np.float32), np.zeros((1, 3, ch), np.float32))]
    st, scan = hqlib.States(hk, hv, dk, dv, 4, 1, None, d[4]), hqlib.Scan(1, T)
    scan.set(st, [T], [-1], [-1])
    for eps in (1e-6, 1e-38):
        out = hqlib.DevBuf.from_array(np.full((T, ch), np.nan, np.float16))
        hqlib.delta_append(scan, st, d[0], d[1], d[2], d[2], d[3], d[3], out, hqlib.DevBuf(T * 4), hqlib.DevBuf(T * 4), f32=True, eps=eps)
        hqlib.synchronize()
        y = out.download((T, ch), np.float16)
        assert (y[:, :dk] == 0).all() and np.isfinite(y).all() and (np.abs(y[:, dk:2 * dk].astype(np.float64) - 1 / 8) < 2.0 ** -12).all()
    scan.free()
