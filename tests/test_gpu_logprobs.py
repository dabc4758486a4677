"""hq_logprobs against float64 log-softmax: vocabularies around every vector and workgroup width, barred tokens, rows of
nothing, infinities, NaN, ties, misaligned rows.

Bounds: an fp32 sum of V exponentials, each within 2^-21, in chains of at most V / 64 + 64 additions; a log probability adds
the roundings of its own terms, the entropy those of sum p |x - max| too. Token numbers are exact."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24


def reference(x, ids, k):
    x = x.astype(np.float64)
    M, V = x.shape
    m = x.max(1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        z = np.exp(x - m).sum(1, keepdims=True)
        lp = np.where(m == -np.inf, -np.inf, x - m - np.log(z))
        d = np.where(x == -np.inf, 0, x - m)
        p = np.exp(x - m) / z
        ent = np.where(m[:, 0] == -np.inf, 0, np.log(z[:, 0]) - (p * d).sum(1))
        spread = (p * np.abs(d)).sum(1)
    bad = np.isnan(x).any(1) | (x == np.inf).any(1)
    lp[bad], ent[bad] = np.nan, np.nan
    with np.errstate(over="ignore"):
        lp = lp.astype(np.float32).astype(np.float64)  # what an fp32 output can hold: -6.8e38 is -inf
    logp = np.stack([[lp[r, i] if i < V else np.nan for i in ids[r]] for r in range(M)])
    rank = np.where(np.isnan(x), np.inf, x)
    top = np.stack([np.lexsort((np.arange(V), -rank[r], ~np.isnan(x[r])))[:k] for r in range(M)])
    return logp, ent, top, np.take_along_axis(lp, top, 1), spread


def check(hq, x, ids, k, shift=0, pad=0):
    M, V = x.shape
    f32 = x.dtype == np.float32
    wide = np.full((M, V + pad), 9999, x.dtype)
    wide[:, :V] = x
    flat = np.concatenate([np.full(shift, 9999, x.dtype), wide.reshape(-1)])
    dx, di = hq.DevBuf.from_array(flat), hq.DevBuf.from_array(ids.astype(np.uint32))
    n = ids.shape[1]
    out = [hq.DevBuf.from_array(np.full(s, 7, np.float32)) for s in (M * n, M, M * max(k, 1), M * max(k, 1))]
    print(f"[gpu] logprobs {M} x {V} {x.dtype} k={k} shift={shift} pad={pad}", flush=True)
    hq.logprobs(dx.ptr + shift * x.itemsize, M, V, f32=f32, stride=V + pad, ids=di, n_ids=n, top_k=k, logp=out[0], entropy=out[1],
                top_ids=out[2] if k else None, top_logp=out[3] if k else None)
    hq.synchronize()
    logp, ent, top, top_logp, spread = reference(x, ids, k)
    E = (V / 64 + 64) * U32 + 2.0 ** -21

    def close(got, want, tol):
        assert np.array_equal(np.isnan(got), np.isnan(want)), (got, want)
        with np.errstate(invalid="ignore"):
            bad = ~((np.abs(got - want) <= tol) | (got == want) | np.isnan(want))
        assert not bad.any(), (got[bad][:4], want[bad][:4])

    close(out[0].download((M, n), np.float32), logp, E + 4 * U32 * np.abs(np.nan_to_num(logp, neginf=0)))
    with np.errstate(invalid="ignore"):
        close(out[1].download((M,), np.float32), ent, E * (2 + 3 * spread) + 4 * U32 * np.abs(ent))
    if k:
        assert np.array_equal(out[2].download((M, k), np.uint32), top)
        close(out[3].download((M, k), np.float32), top_logp, E + 4 * U32 * np.abs(np.nan_to_num(top_logp, neginf=0)))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("M,V,k,n", [(1, 1, 1, 1), (3, 2, 2, 2), (2, 63, 5, 3), (5, 64, 64, 1), (2, 65, 20, 1), (1, 255, 64, 8), (4, 1000, 0, 1),
                                     (3, 4097, 20, 4), (70, 2049, 5, 2), (1, 32000, 5, 4), (17, 32000, 64, 1), (300, 1777, 1, 1), (1, 151936, 20, 1),
                                     (33, 151936, 20, 2), (600, 5000, 3, 1)])
def test_logprobs(hqlib, M, V, k, n, dtype):
    rng = np.random.default_rng(V + M)
    x = (rng.normal(0, 3, (M, V)) + 12 * (rng.random((M, V)) < 4 / V)).astype(dtype)
    check(hqlib, x, rng.integers(0, V, (M, n)), k)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("V,shift,pad", [(1000, 1, 0), (1001, 0, 0), (32001, 3, 6), (4096, 5, 3), (64, 7, 1)])
def test_rows_off_alignment(hqlib, V, shift, pad, dtype):
    rng = np.random.default_rng(V + shift)
    check(hqlib, rng.normal(0, 2, (5, V)).astype(dtype), rng.integers(0, V, (5, 2)), 9, shift, pad)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("V", [70, 3000, 40000])
def test_barred_tokens_ties_and_odd_values(hqlib, V, dtype):
    rng = np.random.default_rng(V)
    big = np.finfo(dtype).max
    rows = []
    for kind in range(14):
        x = rng.normal(0, 1, V).astype(dtype)
        if kind == 0:
            x[rng.random(V) < 0.9] = -np.inf
        elif kind == 1:
            x[:] = -np.inf
        elif kind == 2:
            x[:] = -np.inf
            x[V - 1] = -3
        elif kind == 3:
            x[:] = 0.5
        elif kind == 4:
            x = rng.integers(0, 3, V).astype(dtype)
        elif kind == 5:
            x[V // 2] = np.nan
            x[V - 1] = np.inf
            x[3] = np.nan
        elif kind == 6:
            x[7] = np.inf
        elif kind == 7:
            x[:] = -big
        elif kind == 8:
            x[:] = -big
            x[V - 2] = -np.inf
            x[5] = 0
        elif kind == 9:
            x[::2], x[1::2] = 0.0, -0.0
        elif kind == 10:
            x = np.sort(x)
        elif kind == 11:
            x = np.sort(x)[::-1]
        elif kind == 12:
            x[:] = big
        elif kind == 13:
            x[:] = -big
            x[11] = big
        rows.append(x)
    x = np.stack(rows)
    ids = rng.integers(0, V, (len(x), 4))
    ids[:, 3] = [V, V + 5, 2 ** 32 - 1, V - 1] * 3 + [0, V]
    for k in (1, 33, 64):
        check(hqlib, x, ids, k)


def test_streams_and_missing_outputs(hqlib):
    """Two streams at once, each with a workspace of its own, and only some outputs asked for."""
    rng = np.random.default_rng(2)
    V = 50000
    sts = [hqlib.Stream(), hqlib.Stream()]
    xs = [rng.normal(0, 3, (m, V)).astype(np.float32) for m in (2, 3)]
    dev = [hqlib.DevBuf.from_array(x) for x in xs]
    top = [hqlib.DevBuf(4 * 3 * 8) for _ in xs]
    ent = hqlib.DevBuf(12)
    for _ in range(5):
        for x, d, t, s in zip(xs, dev, top, sts):
            hqlib.logprobs(d, len(x), V, f32=True, top_k=8, top_ids=t, stream=s.ptr)
    hqlib.logprobs(dev[1], 3, V, f32=True, entropy=ent, stream=sts[0].ptr)
    hqlib.synchronize()
    for x, t in zip(xs, top):
        assert np.array_equal(t.download((len(x), 8), np.uint32), np.argsort(-x, 1, kind="stable")[:, :8])
    p = np.exp(xs[1].astype(np.float64))
    p /= p.sum(1, keepdims=True)
    assert np.allclose(ent.download((3,), np.float32), -(p * np.log(p)).sum(1), rtol=1e-4)
    for s in sts:
        s.destroy()


def test_refusals(hqlib):
    b = hqlib.DevBuf(4096)
    for a, kw, msg in (((b, -1, 10), {}, "-1 rows"), ((b, 1, 0), {}, "1 rows of 0"), ((b, 1, 10), dict(stride=9), "stride 9"), ((b, 1, 10), dict(top_k=11), "top_k 11"),
                       ((b, 1, 100), dict(top_k=65), "top_k 65"), ((b, 1, 10), dict(n_ids=-1), "-1 tokens"), ((None, 1, 10), dict(entropy=b), "null"),
                       ((b, 1, 10), dict(n_ids=1, logp=b), "null"), ((b.ptr + 2, 1, 10), dict(entropy=b), "misaligned")):
        with pytest.raises(hqlib.HQError, match=msg):
            hqlib.logprobs(*a, f32=True, **kw)
    hqlib.logprobs(None, 0, 10, f32=True, entropy=b)  # no rows: nothing to do
