"""Calls of more rows than the threads of one launch (2^32) take, at the ends of what the header allows."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def fill(hqlib, buf, block):
    """buf: block again and again (its first copy from the host, the others on the device)."""
    buf.upload(block)
    at = block.nbytes
    while at < buf.nbytes:
        n = min(at, buf.nbytes - at)
        assert hqlib.load().hq_memcpy_d2d(buf.ptr + at, buf.ptr, n, None) == 0
        at += n


def test_delta_single_tokens_of_many_sequences(hqlib):
    """One token of each of 8200 sequences that begin, 1024 heads of 16 x 256: o = scale (q k) beta v. 8.4 million heads of eight waves."""
    n, hv, dk, dv = 8200, 1024, 16, 256
    print(f"[gpu] delta {n} single tokens, {hv} heads", flush=True)
    rng = np.random.default_rng(1)
    rows = 8  # (the values repeat every 8 tokens, everything else is each token's own)
    v = rng.normal(0, 1, (rows, hv, dv)).astype(np.float16)
    qk = rng.normal(0, 0.2, (n, 2 * dk)).astype(np.float16)
    beta = rng.uniform(0, 1, (n, hv)).astype(np.float32)
    d_v, out = hqlib.DevBuf(n * hv * dv * 2), hqlib.DevBuf(n * hv * dv * 2)
    fill(hqlib, d_v, v)
    fill(hqlib, out, np.full(1 << 20, 7, np.float16))
    d_qk, d_beta, d_g, state = hqlib.DevBuf.from_array(qk), hqlib.DevBuf.from_array(beta), hqlib.DevBuf.from_array(np.zeros((n, hv), np.float32)), hqlib.DevBuf(hv * dk * dv * 4)
    st = hqlib.States(1, hv, dk, dv, 1, 1, state, None)
    scan = hqlib.Scan(n, n)
    scan.set(st, [1] * n, [-1] * n, [-1] * n)
    hqlib.delta(scan, st, d_qk, d_qk.ptr + 2 * dk, d_v, d_g, d_beta, out, 1.0, qk_stride=2 * dk, v_stride=hv * dv)
    hqlib.synchronize()
    kq = (qk[:, :dk].astype(np.float64) * qk[:, dk:].astype(np.float64)).sum(-1)
    mag = np.abs(qk[:, :dk].astype(np.float64) * qk[:, dk:].astype(np.float64)).sum(-1)
    for t in (*range(0, 8), 4000, 8190, 8191, 8192, 8193, *range(8194, 8200)):
        y = out.download((hv, dv), np.float16, offset=t * hv * dv * 2).astype(np.float64)
        u = beta[t][:, None].astype(np.float64) * v[t % rows].astype(np.float64)
        # (sums of 16 products and three more operations in 32 bits, then fp16)
        assert (np.abs(y - kq[t] * u) <= (20 * 2.0 ** -24 * mag[t] + 2.0 ** -11 * abs(kq[t])) * np.abs(u) + 2.0 ** -25).all(), t
    scan.free()
