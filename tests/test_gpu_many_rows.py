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


ROWS = (1 << 23) + 5  # of 512 threads: 2^32 and more


def logits(V):
    """Multiples of 1/8 in falling and rising order, unlike from row to row."""
    r = np.arange(ROWS, dtype=np.int64)[:, None]
    return (((r * 7 + np.arange(V) * 5 * (1 + r % 3)) % 64) / 8.0).astype(np.float32)


def test_logprobs_of_many_rows(hqlib):
    print(f"[gpu] logprobs of {ROWS} rows", flush=True)
    V = 3
    x = logits(V)
    d = hqlib.DevBuf.from_array(x)
    ids = hqlib.DevBuf.from_array((np.arange(ROWS) % V).astype(np.uint32))
    out = [hqlib.DevBuf.from_array(np.full(ROWS + 1, 77, np.uint32)) for _ in range(4)]
    hqlib.logprobs(d, ROWS, V, f32=True, ids=ids, n_ids=1, top_k=1, logp=out[0], entropy=out[1], top_ids=out[2], top_logp=out[3])
    hqlib.synchronize()
    got = [o.download(ROWS + 1, t) for o, t in zip(out, (np.float32, np.float32, np.uint32, np.float32))]
    assert all(g.view(np.uint32)[-1] == 77 for g in got)
    e = x.astype(np.float64) - x.max(-1, keepdims=True)
    lp = e - np.log(np.exp(e).sum(-1, keepdims=True))
    r = np.arange(ROWS)
    # (three exponentials and a logarithm in 32 bits, of values up to 8 + log 3)
    assert np.abs(got[0][:-1] - lp[r, r % V]).max() <= 2.0 ** -18 and np.abs(got[3][:-1] - lp.max(-1)).max() <= 2.0 ** -18
    assert np.abs(got[1][:-1] + (np.exp(lp) * lp).sum(-1)).max() <= 2.0 ** -18
    assert np.array_equal(got[2][:-1], x.argmax(-1))


@pytest.mark.parametrize("beams", [1, 3])
def test_beams_of_many_groups(hqlib, beams):
    print(f"[gpu] beams of {ROWS} rows in groups of {beams}", flush=True)
    V, k, G = 3, 2, ROWS // beams
    x = logits(V)[:G * beams]
    rng = np.random.default_rng(beams)
    score = rng.integers(-40, 0, G * beams).astype(np.float32) / 16
    done = (rng.random(G * beams) < 0.1).astype(np.uint8)
    d = [hqlib.DevBuf.from_array(a) for a in (x, score, done)]
    out = [hqlib.DevBuf.from_array(np.full(G * k + 1, 77, np.uint32)) for _ in range(3)]
    hqlib.beam(d[0], G, beams, V, d[1], k, *out, f32=True, done=d[2], done_token=9)
    hqlib.synchronize()
    got = [o.download(G * k + 1, t) for o, t in zip(out, (np.float32, np.uint32, np.int32))]
    assert all(g.view(np.uint32)[-1] == 77 for g in got)
    e = x.astype(np.float64) - x.max(-1, keepdims=True)
    val = score[:, None].astype(np.float64) + (e - np.log(np.exp(e).sum(-1, keepdims=True)))
    tok = np.broadcast_to(np.arange(V), val.shape).copy()
    val[done != 0, 1:], val[done != 0, 0], tok[done != 0] = -np.inf, score[done != 0], 9
    val, tok = val.reshape(G, beams * V), tok.reshape(G, beams * V)
    at = np.argsort(-val, axis=1, kind="stable")[:, :k + 1]
    best = np.take_along_axis(val, at, 1)
    score_got, token_got, beam_got = (g[:-1].reshape(G, k) for g in got)
    some = np.isfinite(best[:, :k])
    with np.errstate(invalid="ignore"):
        assert (np.where(some, np.abs(score_got - best[:, :k]), 0) <= 2.0 ** -19).all() and (score_got[~some] == -np.inf).all()
        # choices where no other value is near (values of unlike rows are off by 2^-20 each)
        clear = some & (np.nan_to_num(best[:, :k] - best[:, 1:], posinf=1) > 2.0 ** -19)
    clear = np.logical_and.accumulate(clear, 1)
    assert clear.mean() > 0.5
    assert (token_got == np.take_along_axis(tok, at, 1)[:, :k])[clear].all() and (beam_got == at[:, :k] // V)[clear].all()
    assert (beam_got[~some] == -1).all() and (token_got[~some] == 0xffffffff).all()


def test_append_of_many_tokens(hqlib):
    """2^24 tokens of one sequence, not rotated: the cache's pages have the keys and values, the queries are as they were."""
    n, d, page = 1 << 24, 16, 4096
    print(f"[gpu] append of {n} tokens", flush=True)
    rng = np.random.default_rng(2)
    block = rng.normal(0, 1, (3, 1 << 13, d)).astype(np.float16)  # (the values repeat every 2^13 tokens)
    q, k, v = (hqlib.DevBuf(n * d * 2) for _ in range(3))
    for buf, b in zip((q, k, v), block):
        fill(hqlib, buf, b)
    q_out, ck, cv = (hqlib.DevBuf(n * d * 2) for _ in range(3))
    for buf in (q_out, ck, cv):
        fill(hqlib, buf, np.full(1 << 16, np.nan, np.float16))
    kv = hqlib.KvCache(hqlib.KV_F16, n // page, page, 1, d, ck, cv, (page * d, d, d))
    pages = rng.permutation(n // page).astype(np.uint32)
    batch = hqlib.Batch(1, n, n // page)
    batch.set(kv, 1, [n], [n], pages[None])
    hqlib.rope_append(batch, kv, q, k, v, q_out, None, 0, 0, f32=False, q_stride=d, kv_stride=d)
    hqlib.synchronize()
    for p in (*range(0, n // page, 97), n // page // 2 - 1, n // page // 2, n // page - 1):
        want = block[:, p * page % (1 << 13):][:, :page]
        at = int(pages[p]) * page * d * 2
        assert np.array_equal(q_out.download((page, d), np.float16, offset=p * page * d * 2), want[0]), p
        assert np.array_equal(ck.download((page, d), np.float16, offset=at), want[1]) and np.array_equal(cv.download((page, d), np.float16, offset=at), want[2]), p
    batch.free()


def test_attention_of_many_sequences(hqlib):
    """2^20 sequences of one token and 16 heads, which all read one page: each has the values of its one position."""
    n, heads, d, page = 1 << 20, 16, 16, 16
    print(f"[gpu] attention of {n} sequences", flush=True)
    rng = np.random.default_rng(3)
    c = rng.normal(0, 1, (2, page, heads, d)).astype(np.float16)
    c[:, 1:] = np.nan
    kv = hqlib.KvCache(hqlib.KV_F16, 1, page, heads, d, *(hqlib.DevBuf.from_array(a) for a in c), (page * heads * d, heads * d, d))
    q, out = hqlib.DevBuf(n * heads * d * 2), hqlib.DevBuf(n * heads * d * 2)
    fill(hqlib, q, rng.normal(0, 1, (1 << 10, heads, d)).astype(np.float16))
    fill(hqlib, out, np.full(1 << 16, np.nan, np.float16))
    batch = hqlib.Batch(n, n, 1)
    batch.set(kv, heads, np.ones(n, np.int32), np.ones(n, np.int32), np.zeros((n, 1), np.uint32))
    hqlib.attention(batch, kv, q, out, 0.25)
    hqlib.synchronize()
    y = out.download((n, heads, d), np.float16)
    assert (y == c[1, 0]).all()
    batch.free()


@pytest.mark.parametrize("f32", [True, False])
def test_longest_rows(hqlib, f32):
    """One row of 2^30 logits, the likeliest at its ends and on both sides of 4 GB: hq_beam's values to 2^-20, hq_logprobs' to what sums of 2^16
    terms in 32 bits each lose (2^-24 a sum, at most 2^16 of them in a row: 2^-8)."""
    V, t = 1 << 30, np.float32 if f32 else np.float16
    print(f"[gpu] rows of {V}, f32={f32}", flush=True)
    block = (np.random.default_rng(4).integers(-64, 0, 1 << 20) / 16.0).astype(t)
    row = hqlib.DevBuf(V * block.itemsize)
    fill(hqlib, row, block)
    top = {V - 1: 5.0, 0: 4.0, V // 2: 3.0, V // 2 - 1: 3.0, (1 << 29) + 12345: 2.0, V - 2: 1.5, 777: 1.0, V - 100000: 0.5}
    total = np.exp(block.astype(np.float64)).sum() * (V / len(block))
    for i, x in top.items():
        row.upload(np.array([x], t), offset=i * block.itemsize)
        total += np.exp(x) - np.exp(float(block[i % len(block)]))
    order = sorted(top, key=lambda i: (-top[i], i))
    k = len(order)
    want = np.array([top[i] for i in order]) - np.log(total)
    score = hqlib.DevBuf.from_array(np.array([-0.5], np.float32))
    out = [hqlib.DevBuf(k * 4) for _ in range(5)]
    hqlib.beam(row, 1, 1, V, score, k, *out[:3], f32=f32)
    hqlib.logprobs(row, 1, V, f32=f32, top_k=k, top_ids=out[3], top_logp=out[4])
    hqlib.synchronize()
    assert out[1].download(k, np.uint32).tolist() == order and out[3].download(k, np.uint32).tolist() == order
    assert np.abs(out[0].download(k, np.float32) - (want - 0.5)).max() <= 2.0 ** -19 + 2.0 ** -24 * 32
    assert np.abs(out[4].download(k, np.float32) - want).max() <= 2.0 ** -8
