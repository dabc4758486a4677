"""hq_rope_append and hq_rope_table against float64 (tests/serve_ref.py), at the edges of head sizes, pages and positions.

Bound of a stored value: its rounding to fp16 (2^-11 of it, 2^-25 where subnormal) and some ten fp32 roundings of what it is
made of; with RMSNorm a sum of hd squares more, hd 2^-24 relative at most. Q8: half a code, the scale's rounding to fp16."""
import numpy as np
import pytest

from serve_ref import U16, U32, Pool, rope

pytestmark = pytest.mark.gpu

# heads, kv heads, head_dim, rot, f32, norm, axes, page, layout, q8, (new, total) of each sequence
CASES = [
    (8, 8, 64, 64, True, False, 1, 16, "pos", False, [(1, 1)]),
    (8, 8, 64, 64, False, True, 1, 16, "head", True, [(17, 33), (1, 16), (0, 5), (3, 3)]),
    (32, 8, 128, 128, True, True, 1, 64, "pos", False, [(1, 1000), (1, 64), (1, 65), (70, 70), (5, 2), (2, 0)]),
    (4, 2, 80, 40, True, False, 1, 32, "pos", True, [(40, 100), (1, 7)]),
    (3, 1, 96, 96, False, True, 3, 128, "head", False, [(130, 131), (2, 300)]),
    (16, 4, 256, 64, False, True, 3, 256, "pos", True, [(33, 600), (1, 1)]),
    (2, 1, 16, 16, True, False, 1, 16, "head", True, [(20, 20)]),
    (5, 5, 48, 0, True, False, 1, 16, "pos", False, [(9, 40)]),
    (64, 8, 128, 128, True, False, 1, 4096, "pos", False, [(300, 5000)]),
    (4, 1, 240, 8, True, True, 1, 64, "head", False, [(19, 64)]),
]


def put_rows(hq, rng, T, nh, nkv, hd, f32, gated):
    """[q (| gate) per head | k | v] rows of one product with eight values of other use at the end of each."""
    per = 2 * hd if gated else hd
    x = rng.normal(0, 2, (T, nh * per + 2 * nkv * hd + 8)).astype(np.float32 if f32 else np.float16)
    q = x[:, :nh * per].reshape(T, nh, per)[:, :, :hd]
    k = x[:, nh * per:nh * per + nkv * hd].reshape(T, nkv, hd)
    v = x[:, nh * per + nkv * hd:nh * per + 2 * nkv * hd].reshape(T, nkv, hd)
    return x, q, k, v, per


@pytest.mark.parametrize("nh,nkv,hd,rot,f32,norm,axes,page,layout,q8,lens", CASES)
def test_rope_append(hqlib, nh, nkv, hd, rot, f32, norm, axes, page, layout, q8, lens):
    rng = np.random.default_rng(nh * hd + page)
    n_new, n_pos = [a for a, _ in lens], [b for _, b in lens]
    T, gated = sum(n_new), nh % 2 == 0
    x, q, k, v, per = put_rows(hqlib, rng, T, nh, nkv, hd, f32, gated)
    pool = Pool(rng, n_pos, page, nkv, hd, q8, layout)
    kv = pool.device(hqlib)
    b = hqlib.Batch(len(lens), T, pool.table.shape[1])
    b.set(kv, nh, n_new, n_pos, pool.table)
    own = np.concatenate([np.arange(p - n, p) for n, p in lens])
    n_table = max(1, int(own.max()) + 1) if axes == 1 else 50
    inv = (10000.0 ** (-np.arange(rot // 2) * 2 / max(rot, 1))).astype(np.float32)
    table = hqlib.DevBuf(n_table * max(rot // 2, 1) * 8)
    if rot:
        hqlib.rope_table(inv, n_table, table)
    cs = table.download((n_table, rot // 2, 2), np.float32)
    ang = np.arange(n_table)[:, None] * inv.astype(np.float64)
    assert np.abs(cs[..., 0] - np.cos(ang)).max(initial=0) <= 2.0 ** -24 and np.abs(cs[..., 1] - np.sin(ang)).max(initial=0) <= 2.0 ** -24
    axis = rng.integers(0, axes, rot // 2).astype(np.uint8)
    pos = own[None] if axes == 1 else rng.integers(0, n_table, (axes, T)).astype(np.int32)
    w = (1 + 0.1 * rng.normal(0, 1, (2, hd))).astype(np.float32) if norm else [None, None]
    wd = [hqlib.DevBuf.from_array(a) if norm else None for a in w]
    dx = hqlib.DevBuf.from_array(x)
    dp = hqlib.DevBuf.from_array(pos.astype(np.int32)) if axes > 1 else None
    out = hqlib.DevBuf(T * nh * hd * 2)
    size = x.itemsize
    print(f"[gpu] rope_append {nh}/{nkv} x {hd} rot {rot} {lens} q8={q8}", flush=True)
    hqlib.rope_append(b, kv, dx, dx.ptr + nh * per * size, dx.ptr + (nh * per + nkv * hd) * size, out, table if rot else None, n_table, rot,
                      f32=f32, q_stride=x.shape[1], q_head_stride=per, kv_stride=x.shape[1], positions=dp, axis=axis if axes > 1 else None,
                      q_norm=wd[0], k_norm=wd[1], norm_offset=0.25, eps=1e-5)
    hqlib.synchronize()
    sel = pos[axis] if axes > 1 else np.broadcast_to(own, (rot // 2, T))
    turn = cs[np.maximum(sel.T, 0), np.arange(rot // 2)]
    pad = own < 0
    fp = (12 + (hd if norm else 0)) * U32
    y, mag = rope(q, w[0], turn, rot, 0.25, 1e-5)
    y[pad], mag[pad] = 0, 0
    got = out.download((T, nh, hd), np.float16).astype(np.float64)
    assert (np.abs(got - y) <= U16 * np.abs(y) + fp * mag + 2.0 ** -25).all()
    before = {n: pool.c[n].copy() for n in "kv"}
    scales = {n: pool.d[n].copy() for n in "kv"} if q8 else None
    pool.read(hqlib, kv)
    want = {"k": rope(k, w[1], turn, rot, 0.25, 1e-5), "v": (v.astype(np.float64), np.abs(v.astype(np.float64)))}
    seq = np.repeat(np.arange(len(lens)), n_new)
    pg, sl = pool.table[seq[~pad], own[~pad] // page], own[~pad] % page
    for n, (y, mag) in want.items():
        y, mag = y[~pad], mag[~pad]
        at = (pg, sl) if layout == "pos" else (pg, slice(None), sl)
        new = pool.c[n][at]
        if q8:
            d = pool.d[n][pg, :, sl].astype(np.float64)
            top = np.abs(y).max(-1)
            assert (np.abs(d - top / 127) <= (U16 + 2 * fp) * top / 127 + 2.0 ** -25).all()
            assert (np.abs(new * d[..., None] - y) <= 0.5 * d[..., None] + 2 * fp * (mag + top[..., None])).all()
            assert np.abs(new.astype(int)).max() <= 127
            scales[n][pg, :, sl] = pool.d[n][pg, :, sl]
            assert np.array_equal(scales[n].view(np.uint16), pool.d[n].view(np.uint16))
        else:
            assert (np.abs(new.astype(np.float64) - y) <= U16 * np.abs(y) + fp * mag + 2.0 ** -25).all()
        before[n][at] = new  # and nothing else was written
        assert np.array_equal(before[n].view(np.uint8), pool.c[n].view(np.uint8))
    b.free()


def test_values_without_a_number(hqlib):
    """Positions outside the table give NaN in the rotated dims of that token alone; an infinity or NaN makes its own head
    of a Q8 cache NaN, a head of zeros gives zeros."""
    rng = np.random.default_rng(4)
    nh, nkv, hd, T, page = 2, 2, 32, 6, 16
    for q8 in (False, True):
        pool = Pool(rng, [T], page, nkv, hd, q8)
        kv = pool.device(hqlib)
        b = hqlib.Batch(1, T, 1)
        b.set(kv, nh, [T], [T], pool.table)
        x = rng.normal(0, 1, (T, (nh + 2 * nkv) * hd)).astype(np.float32)
        x[3, nh * hd + 5], x[4, (nh + nkv) * hd + 31], x[5, (nh + nkv) * hd:] = np.nan, -np.inf, 0
        table = hqlib.DevBuf(3 * 8 * 8)
        hqlib.rope_table(np.ones(8, np.float32), 3, table)
        pos = hqlib.DevBuf.from_array(np.array([[0, -1, 3, 1, 2, 1 << 30]], np.int32))
        dx, out = hqlib.DevBuf.from_array(x), hqlib.DevBuf(T * nh * hd * 2)
        hqlib.rope_append(b, kv, dx, dx.ptr + nh * hd * 4, dx.ptr + (nh + nkv) * hd * 4, out, table, 3, 16, f32=True, q_stride=x.shape[1],
                          kv_stride=x.shape[1], positions=pos, axis=np.zeros(8, np.uint8))
        hqlib.synchronize()
        got = np.isnan(out.download((T, nh, hd), np.float16))
        off = np.array([False, True, True, False, False, True])
        assert got[off][..., :16].all() and not got[off][..., 16:].any() and not got[~off].any()
        pool.read(hqlib, kv)
        k, v = (pool.get(n, 0, T) for n in "kv")
        if q8:
            bad = np.isnan(k).all(-1)
            assert np.array_equal(bad, np.isnan(k).any(-1)) and np.array_equal(bad, np.stack([off | [0, 0, 0, 1, 0, 0], off], 1).astype(bool))
            bad = np.isnan(v)
            assert bad[4, 0].all() and not bad[4, 1].any() and not bad[:4].any()
        else:
            assert np.isnan(k[3, 0, 5]) and np.isnan(k[3]).sum() == 2 and v[4, 0, 31] == -np.inf and np.isfinite(v).sum() == v.size - 1
        assert (v[5] == 0).all()
        b.free()
