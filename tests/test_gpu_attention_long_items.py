"""hq_attention where a workgroup of k_rows takes long runs of positions: its ring of tiles turns many times, page addresses are
formed again every 64 tiles, and most tiles go through the loop without tests. The step's plan leaves a block of rows whole where
there are as many blocks as the chip has places for workgroups (256 CUs, one or two each), so there are that many kv heads here;
they share one head's memory (head_stride 0), which lets the reference be one float64 product."""
import time

import numpy as np
import pytest

from serve_ref import U16, U32, Pool, fill
from test_gpu_paged_attention import check

pytestmark = pytest.mark.gpu

# kv heads, heads per kv head, head_dim, (new, total): 132 tiles of 32 positions and more; blocks of 128 rows, of 256, all widths
CASES = [(512, 1, 64, [(40, 4230)]), (512, 1, 96, [(33, 4200), (40, 2111)]), (512, 2, 128, [(50, 4200)]), (256, 1, 192, [(35, 4225)]),
         (256, 1, 256, [(70, 4200)]), (256, 4, 128, [(45, 4207)]), (256, 3, 80, [(60, 4300)]), (256, 8, 64, [(20, 4200), (1, 77), (20, 2200)])]


def reference(pool, s, q, n, scale):
    """Outputs and bound (serve_ref.attention's) of sequence s's new tokens q [new, heads, hd] over its n positions."""
    new, nh, hd = q.shape
    k, v = pool.get("k", s, n)[:, 0], pool.get("v", s, n)[:, 0]
    q = q.astype(np.float64)
    later = np.arange(n)[None] > np.arange(n - new, n)[:, None]
    y, bound = np.zeros(q.shape), np.zeros(q.shape)
    for h in range(nh):
        x = np.where(later, -np.inf, q[:, h] @ k.T * scale)
        size = np.where(later, 0, np.abs(q[:, h]) @ np.abs(k).T).max(1, keepdims=True)
        p = np.exp(x - x.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        e = ((hd + 8) * U32 + (U16 if pool.q8 else 0)) * size * abs(scale) + 2.0 ** -20
        y[:, h] = p @ v
        bound[:, h] = U16 * np.abs(y[:, h]) + (U16 * (2 if pool.q8 else 1) + 2 * e) * (p @ np.abs(v)) + 2.0 ** -24
    return y, bound


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("nkv,rep,hd,lens", CASES)
def test_long_items(hqlib, nkv, rep, hd, lens, q8):
    rng = np.random.default_rng(nkv + rep + hd)
    n_new, n_pos, nh, T = [a for a, _ in lens], [t for _, t in lens], nkv * rep, sum(a for a, _ in lens)
    pool = Pool(rng, n_pos, 16, 1, hd, q8)
    fill(pool, rng, n_pos)
    dev = [hqlib.DevBuf.from_array(pool.c[n]) for n in "kv"]
    scales = [hqlib.DevBuf.from_array(np.repeat(pool.d[n], nkv, 1)) for n in "kv"] if q8 else [None, None]
    kv = hqlib.KvCache(hqlib.KV_Q8 if q8 else hqlib.KV_F16, pool.n_pages, 16, nkv, hd, *dev, (16 * hd, hd, 0), *scales)
    q = rng.normal(0, 1.5, (T, nh, hd)).astype(np.float16)
    dq, out = hqlib.DevBuf.from_array(q), hqlib.DevBuf(q.nbytes)
    b = hqlib.Batch(len(lens), T, pool.table.shape[1])
    b.set(kv, nh, n_new, n_pos, pool.table)
    print(f"[gpu] long items: {nkv} x {rep} heads of {hd} {lens} q8={q8}", flush=True)
    hqlib.attention(b, kv, dq, out, hd ** -0.5)
    hqlib.synchronize()
    got = out.download(q.shape, np.float16).astype(np.float64)
    heads = np.unique(np.concatenate([np.arange(rep), rng.integers(0, nh, 10), [nh - 1]]))  # (a few of them)
    t = 0
    for s, (new, n) in enumerate(lens):
        check(got[t:t + new][:, heads], *reference(pool, s, q[t:t + new][:, heads], n, hd ** -0.5))
        t += new
    assert np.isfinite(got).all()
    b.free()


@pytest.mark.parametrize("nkv,rep,hd,n", [(256, 8, 128, 660), (256, 8, 96, 660), (256, 4, 256, 660), (512, 4, 64, 660)])
def test_places_behind_the_end_cost_nothing(hqlib, nkv, rep, hd, n):
    """What stands behind a sequence's last position, in the same tile of 32, costs no time: NaN there take as long as zeros. (An
    odd number of tiles, the last one partial; the loop over values that are not finite would take more than twice as long.)"""
    rng = np.random.default_rng(hd)
    new = 32 if hd != 64 else 20
    page, nh = 64, nkv * rep
    pool = Pool(rng, [n], page, 1, hd)
    fill(pool, rng, [n])
    dq, out = hqlib.DevBuf.from_array(rng.normal(0, 1, (new, nh, hd)).astype(np.float16)), hqlib.DevBuf(new * nh * hd * 2)
    kvs = []
    for empty in (np.nan, 0):
        dev = [hqlib.DevBuf.from_array(np.where(np.isnan(pool.c[m]), np.float16(empty), pool.c[m])) for m in "kv"]
        kvs.append(hqlib.KvCache(hqlib.KV_F16, pool.n_pages, page, nkv, hd, *dev, (page * hd, hd, 0)))
    b = hqlib.Batch(1, new, pool.table.shape[1])
    b.set(kvs[0], nh, [new], [n], pool.table)
    print(f"[gpu] places behind the end: {nkv} x {rep} heads of {hd}", flush=True)
    best = [1e9, 1e9]
    for _ in range(12):
        for i, kv in enumerate(kvs):
            hqlib.synchronize()
            t = time.perf_counter()
            for _ in range(20):
                hqlib.attention(b, kv, dq, out, hd ** -0.5)
            hqlib.synchronize()
            best[i] = min(best[i], time.perf_counter() - t)
    print(f"[gpu]   {best[0] / 20 * 1e6:.1f} us, with zeros {best[1] / 20 * 1e6:.1f}", flush=True)
    assert best[0] <= 1.3 * best[1]
    b.free()
