"""hq_attention against float64 softmax attention (tests/serve_ref.py, which derives the bound of each element): tile and
page edges, grouped heads, sequences without tokens or positions, padding, strides, gates, caches past 32-bit offsets,
and places that must not matter holding NaN (every pool's unwritten places do)."""
import numpy as np
import pytest

from serve_ref import Pool, attention, fill

pytestmark = pytest.mark.gpu

# heads, kv heads, head_dim, page, layout, (new, total) of each sequence
CASES = [
    (8, 8, 64, 16, "pos", [(1, 1)]),
    (8, 8, 64, 16, "head", [(1, 1001), (1, 15), (1, 16), (1, 17), (0, 40), (1, 0), (0, 0)]),
    (32, 8, 128, 64, "pos", [(1, 31), (1, 32), (1, 33), (1, 63), (1, 64), (1, 65), (1, 500), (1, 2)]),
    (16, 2, 128, 32, "head", [(1, 900), (2, 129), (3, 3), (5, 64), (4, 200)]),
    (4, 4, 80, 128, "pos", [(33, 33), (1, 130), (17, 90)]),
    (6, 2, 96, 16, "head", [(70, 100), (65, 65), (3, 2), (40, 7)]),
    (16, 4, 256, 64, "pos", [(1, 300), (40, 130), (9, 64)]),
    (8, 1, 240, 32, "head", [(20, 50), (1, 70)]),
    (2, 1, 16, 16, "pos", [(100, 100), (1, 333)]),
    (3, 1, 48, 256, "head", [(130, 257), (1, 256)]),
    (64, 1, 64, 16, "pos", [(1, 100), (3, 40)]),
    (5, 5, 112, 512, "pos", [(64, 64), (63, 127), (1, 1), (129, 300)]),
    (40, 8, 128, 64, "pos", [(30, 30), (31, 200)]),
    (2, 2, 128, 64, "head", [(1, 5000), (256, 600)]),
    (1, 1, 192, 16, "pos", [(300, 300)]),
]


def run(hq, pool, nh, lens, q, scale, stream=None, gate=None, gate_f32=False, pad=0, **kw):
    T, hd = q.shape[0], pool.hd
    kv = pool.device(hq)
    b = hq.Batch(len(lens), T, pool.table.shape[1])
    b.set(kv, nh, [a for a, _ in lens], [t for _, t in lens], pool.table, stream)
    wide = np.zeros((T, nh * hd + pad), np.float16)
    wide[:, :nh * hd] = q.reshape(T, -1)
    dq, out = hq.DevBuf.from_array(wide), hq.DevBuf.from_array(np.full((T, nh * hd + 2 * pad), 7, np.float16))
    g = {}
    if gate is not None:  # [T, nh, 2 hd] rows whose second halves are the gate
        both = np.concatenate([np.full_like(gate, np.nan), gate], -1).astype(np.float32 if gate_f32 else np.float16)
        dg = hq.DevBuf.from_array(both)
        g = dict(gate=dg.ptr + hd * both.itemsize, gate_f32=gate_f32, gate_stride=2 * nh * hd, gate_head_stride=2 * hd)
    res = []
    for _ in range(2):
        hq.attention(b, kv, dq, out, scale, q_stride=wide.shape[1], out_stride=nh * hd + 2 * pad, stream=stream, **g)
        hq.synchronize()
        res.append(out.download((T, nh * hd + 2 * pad), np.float16))
    assert np.array_equal(res[0].view(np.uint16), res[1].view(np.uint16)), "two calls differ"
    assert (res[0][:, nh * hd:] == 7).all()
    b.free()
    return res[0][:, :nh * hd].reshape(T, nh, hd).astype(np.float64)


def check(got, want, bound):
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    with np.errstate(invalid="ignore"):
        bad = ~((np.abs(got - want) <= bound) | (got == want)) & ok
    worst = np.nanmax(np.where(bad, np.abs(got - want) / bound, 0)) if bad.any() else 0
    assert not bad.any(), (int(bad.sum()), worst, np.argwhere(bad)[:4])


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("nh,nkv,hd,page,layout,lens", CASES)
def test_attention(hqlib, nh, nkv, hd, page, layout, lens, q8):
    rng = np.random.default_rng(nh + hd + page)
    n_new, n_pos = [a for a, _ in lens], [t for _, t in lens]
    pool = Pool(rng, n_pos, page, nkv, hd, q8, layout)
    fill(pool, rng, n_pos)
    q = rng.normal(0, 2, (sum(n_new), nh, hd)).astype(np.float16)
    print(f"[gpu] attention {nh}/{nkv} x {hd} page {page} {lens} q8={q8}", flush=True)
    got = run(hqlib, pool, nh, lens, q, hd ** -0.5)
    check(got, *attention(pool, q, n_new, n_pos, hd ** -0.5))


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("hd", [16, 48, 64, 80, 96, 112, 128, 160, 192, 256])
def test_blocks_cut_into_parts(hqlib, hd, q8):
    """Long sequences with few rows, whose positions go to several workgroups: rows of 16, of 32, of 128 and 256, every
    width of the kernels; a part's rows must fit the workspace that the plan gave them."""
    rng = np.random.default_rng(hd)
    for nh, lens in ((1, [(1, 4000), (20, 3500)]), (2, [(1, 9), (1, 6000), (1, 33), (40, 3000)]), (4, [(130, 2048)])):
        pool = Pool(rng, [t for _, t in lens], 64, 1, hd, q8)
        fill(pool, rng, [t for _, t in lens])
        q = rng.normal(0, 1.5, (sum(a for a, _ in lens), nh, hd)).astype(np.float16)
        print(f"[gpu] parts: {nh} heads x {hd} {lens} q8={q8}", flush=True)
        got = run(hqlib, pool, nh, lens, q, hd ** -0.5)
        check(got, *attention(pool, q, [a for a, _ in lens], [t for _, t in lens], hd ** -0.5))


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("nh,hd,lens", [(1, 64, [(1, 40000)]), (16, 128, [(1, 20000), (1, 3)]), (24, 64, [(1, 20000), (16, 16), (0, 5)]), (9, 256, [(1, 30000)]),
                                        (20, 128, [(1, 300), (2, 9000)]), (4, 64, [(100, 500), (20, 3000), (1, 700)])])
def test_many_parts_and_shared_kernels(hqlib, nh, hd, lens, gate):
    """One kv head behind up to 128 parts a block, more than a wave's lanes; 16 and 32 rows, and 128 and 256, in one step."""
    rng = np.random.default_rng(nh + hd)
    pool = Pool(rng, [t for _, t in lens], 64, 1, hd, False)
    fill(pool, rng, [t for _, t in lens])
    T = sum(a for a, _ in lens)
    q = rng.normal(0, 1.5, (T, nh, hd)).astype(np.float16)
    g = rng.normal(0, 2, (T, nh, hd)).astype(np.float16) if gate else None
    print(f"[gpu] many parts: {nh} heads x {hd} {lens} gate={gate}", flush=True)
    got = run(hqlib, pool, nh, lens, q, hd ** -0.5, gate=g)
    check(got, *attention(pool, q, [a for a, _ in lens], [t for _, t in lens], hd ** -0.5, gate=g))


@pytest.mark.parametrize("gate_f32", [False, True])
@pytest.mark.parametrize("q8", [False, True])
def test_gate_strides_and_stream(hqlib, q8, gate_f32):
    rng = np.random.default_rng(5)
    lens = [(1, 70), (50, 90), (2, 1)]
    pool = Pool(rng, [t for _, t in lens], 32, 2, 64, q8)
    fill(pool, rng, [t for _, t in lens])
    q = rng.normal(0, 2, (53, 6, 64)).astype(np.float16)
    gate = rng.normal(0, 3, (53, 6, 64)).astype(np.float16)
    gate[7, 2, :4], gate[8, 1, 5] = [np.inf, -np.inf, 60000, -60000], 0
    st = hqlib.Stream()
    got = run(hqlib, pool, 6, lens, q, 0.2, st.ptr, gate, gate_f32, pad=24)
    with np.errstate(over="ignore"):
        check(got, *attention(pool, q, [1, 50, 2], [70, 90, 1], 0.2, gate))
    st.destroy()


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("nh,nkv,hd,lens,at", [(4, 2, 64, [(40, 100)], 80), (4, 4, 128, [(3, 40), (70, 70)], 38), (8, 1, 256, [(2, 65)], 64),
                                               (2, 2, 96, [(150, 200)], 130)])
def test_later_positions_do_not_matter(hqlib, q8, nh, nkv, hd, lens, at):
    """A position that only the chunk's later tokens see holds infinities and NaN, in keys, in values, or in one dim of
    them: tokens before it are as if it held numbers, tokens from it on are what the formula gives."""
    rng = np.random.default_rng(hd + at)
    n_new, n_pos = [a for a, _ in lens], [t for _, t in lens]
    pool = Pool(rng, n_pos, 16, nkv, hd, q8)
    fill(pool, rng, n_pos)
    q = rng.normal(0, 1, (sum(n_new), nh, hd)).astype(np.float16)
    first = n_new[0] - (n_pos[0] - at)  # the first token that sees position `at` of sequence 0
    clean, bound = attention(pool, q, n_new, n_pos, 0.1)
    keep = {n: pool.c[n].copy() for n in "kv"}
    scales = {n: pool.d[n].copy() for n in "kv"} if q8 else None
    pg, sl = pool.table[0, at // 16], at % 16
    for name, value in (("v", np.nan), ("k", np.nan), ("v", np.inf), ("k", -np.inf)):
        if q8:
            pool.d[name][pg, :, sl] = value
        else:
            pool.c[name][pg, sl, :, 0 if value == np.inf else slice(None)] = value
        got = run(hqlib, pool, nh, lens, q, 0.1)
        check(got[:first], clean[:first], bound[:first])
        check(got[n_new[0]:], clean[n_new[0]:], bound[n_new[0]:])
        with np.errstate(invalid="ignore"):
            want, b = attention(pool, q, n_new, n_pos, 0.1)
        if name == "v" or np.isnan(value):
            check(got[first:n_new[0]], want[first:n_new[0]], b[first:n_new[0]])
        pool.c = {n: keep[n].copy() for n in "kv"}
        if q8:
            pool.d = {n: scales[n].copy() for n in "kv"}


@pytest.mark.parametrize("std,scale", [(8.0, 0.125), (0.01, 1.0), (60.0, 1.0), (4.0, -0.125), (1.0, 0.0)])
def test_sharp_flat_and_signed_scores(hqlib, std, scale):
    rng = np.random.default_rng(3)
    lens = [(1, 777), (60, 200)]
    for q8 in (False, True):
        pool = Pool(rng, [777, 200], 64, 2, 64, q8)
        fill(pool, rng, [777, 200], 1.0)
        q = rng.normal(0, std, (61, 4, 64)).astype(np.float16)
        check(run(hqlib, pool, 4, lens, q, scale), *attention(pool, q, [1, 60], [777, 200], scale))


@pytest.mark.parametrize("q8", [False, True])
def test_small_and_large_values(hqlib, q8):
    """Values near fp16's ends: weights and sums must not lose them."""
    rng = np.random.default_rng(8)
    lens = [(1, 400), (40, 100)]
    for size in (2.0 ** -12, 3e4):
        pool = Pool(rng, [400, 100], 16, 1, 64, q8)
        for s, n in enumerate((400, 100)):
            pool.put(s, np.arange(n), rng.normal(0, 1, (n, 1, 64)).astype(np.float16), (size * rng.uniform(-1, 1, (n, 1, 64))).astype(np.float16))
        q = rng.normal(0, 1, (41, 2, 64)).astype(np.float16)
        want, bound = attention(pool, q, [1, 40], [400, 100], 0.125)
        # codes of a small scale decode into fp16's subnormal range: half its step more
        check(run(hqlib, pool, 2, lens, q, 0.125), want, bound + (2.0 ** -25 if q8 else 0))


def test_offsets_past_32_bits(hqlib):
    """Pages more than 2^31 elements (4 GiB) apart, as in a cache of tens of GiB."""
    rng = np.random.default_rng(9)
    nkv, hd, page, n = 1, 64, 16, 48
    gap = (1 << 31) + 4096  # elements between pages
    buf = hqlib.DevBuf((4 * gap + (1 << 20)) * 2)
    half = 1 << 17  # values stand half pages' bytes further
    kv = hqlib.KvCache(hqlib.KV_F16, 5, page, nkv, hd, buf, buf.ptr + half * 2, (gap, hd, hd))
    table = np.array([[3, 4, 1]], np.uint32)
    x = rng.normal(0, 1, (2, n, hd)).astype(np.float16)
    for i in range(3):
        for j in range(2):
            buf.upload(x[j, 16 * i:16 * i + 16], offset=(int(table[0, i]) * gap + j * half) * 2)
    pool = Pool(rng, [n], page, nkv, hd)
    pool.put(0, np.arange(n), x[0][:, None], x[1][:, None])
    q = rng.normal(0, 2, (20, 2, hd)).astype(np.float16)
    want, bound = attention(pool, q, [20], [n], 0.125)
    b = hqlib.Batch(1, 20, 3)
    b.set(kv, 2, [20], [n], table)
    dq, out = hqlib.DevBuf.from_array(q), hqlib.DevBuf(q.nbytes)
    hqlib.attention(b, kv, dq, out, 0.125)
    hqlib.synchronize()
    check(out.download(q.shape, np.float16).astype(np.float64), want, bound)
    # and the append's: one more token at the end of the last page
    row = rng.normal(0, 1, (1, 4 * hd)).astype(np.float32)
    dr = hqlib.DevBuf.from_array(row)
    b.set(kv, 2, [1], [n], table)
    hqlib.rope_append(b, kv, dr, dr.ptr + 2 * hd * 4, dr.ptr + 3 * hd * 4, out, None, 0, 0, f32=True, q_stride=4 * hd, kv_stride=4 * hd)
    hqlib.synchronize()
    for j in range(2):
        got = buf.download((hd,), np.float16, offset=(1 * gap + 15 * hd + j * half) * 2)
        assert np.array_equal(got, row[0, (2 + j) * hd:(3 + j) * hd].astype(np.float16))
    b.free(), buf.free()


def test_steps_one_after_another(hqlib):
    """One batch object through prompts, chunks and single tokens; each step appended and attended, positions checked
    against one pass over everything."""
    rng = np.random.default_rng(11)
    nh, nkv, hd, page = 4, 2, 64, 16
    total = [100, 37, 65]
    x = [rng.normal(0, 1, (n, (nh + 2 * nkv) * hd)).astype(np.float32) for n in total]
    pool = Pool(rng, total, page, nkv, hd)
    kv = pool.device(hqlib)
    table = hqlib.DevBuf(128 * 32 * 8)
    hqlib.rope_table((10000.0 ** (-np.arange(32) / 32)).astype(np.float32), 128, table)
    b = hqlib.Batch(3, sum(total), 7)

    def step(new, pos):
        rows = np.concatenate([x[s][p - n:p] for s, (n, p) in enumerate(zip(new, pos))])
        T = len(rows)
        dx, q, out = hqlib.DevBuf.from_array(rows), hqlib.DevBuf(T * nh * hd * 2), hqlib.DevBuf(T * nh * hd * 2)
        b.set(kv, nh, new, pos, pool.table)
        w = rows.shape[1]
        hqlib.rope_append(b, kv, dx, dx.ptr + nh * hd * 4, dx.ptr + (nh + nkv) * hd * 4, q, table, 128, hd, f32=True, q_stride=w, kv_stride=w)
        hqlib.attention(b, kv, q, out, 0.125)
        hqlib.synchronize()
        o = out.download((T, nh, hd), np.float16)
        return np.split(o, np.cumsum(new)[:-1])

    parts = [[], [], []]
    for new, pos in (([50, 37, 0], [50, 37, 0]), ([49, 0, 64], [99, 37, 64]), ([1, 0, 1], [100, 37, 65])):
        for s, o in enumerate(step(new, pos)):
            parts[s].append(o)
    whole = step(total, total)
    for s in range(3):
        got = np.concatenate(parts[s]).astype(np.float64)
        # the same scores in another order of tiles: the fp16 roundings of weights and outputs, twice
        assert np.abs(got - whole[s].astype(np.float64)).max() <= 4 * 2.0 ** -11 * 4
    pool.read(hqlib, kv)
    assert all(np.isfinite(pool.get(n, s, total[s])).all() for n in "kv" for s in range(3))
    b.free()


def test_refusals(hqlib):
    hq = hqlib
    buf = hq.DevBuf(1 << 20)
    f16 = lambda **k: hq.KvCache(k.pop("type", hq.KV_F16), k.pop("n_pages", 8), k.pop("page", 16), k.pop("kv", 2), k.pop("hd", 64),
                                 k.pop("k", buf.ptr), buf.ptr, k.pop("strides", (2048, 128, 64)), **k)
    kv, one = f16(), np.zeros((1, 8), np.uint32)
    for a in ((0, 1, 1), (1, -1, 1), (1, 1, -1)):
        with pytest.raises(hq.HQError, match="hq_batch_create"):
            hq.Batch(*a)
    b = hq.Batch(2, 16, 8)
    with pytest.raises(hq.HQError, match="describes no step"):
        b.n_heads = 2
        hq.attention(b, kv, buf, buf, 1.0)
    for bad, msg in ((f16(type=2), "cache type"), (f16(page=24), "page_size"), (f16(page=8), "page_size"), (f16(hd=72), "head_dim"),
                     (f16(hd=272), "head_dim"), (f16(kv=0), "kv heads"), (f16(n_pages=1 << 28), "2\\^31")):
        with pytest.raises(hq.HQError, match=msg):
            b.set(bad, 2, [1], [1], one)
    for a, msg in (((3, [1], [1], one), "3 heads over 2"), ((2, [1] * 3, [1] * 3, np.zeros((3, 1))), "3 sequences"),
                   ((2, [-1], [1], one), "-1 new tokens"), ((2, [1], [-2], one), "of -2"), ((2, [17], [17], one), "17 new tokens"),
                   ((2, [1], [129], one), "needs 9 pages"), ((2, [1], [17], one[:, :1]), "needs 2 pages"), ((2, [1], [1], one + 8), "page 0 of sequence 0 is 8")):
        with pytest.raises(hq.HQError, match=msg):
            b.set(kv, *a)
        with pytest.raises(hq.HQError, match="describes no step"):
            hq.attention(b, kv, buf, buf, 1.0)
    b.set(kv, 2, [1, 2], [1, 5], np.array([[0], [7]]))
    for bad, msg in ((f16(page=32), "not the one"), (f16(k=None), "no memory"), (f16(k=buf.ptr + 8), "aligned"), (f16(strides=(2048, 128, 24)), "stride 24"),
                     (f16(type=hq.KV_Q8), "not the one")):
        with pytest.raises(hq.HQError, match=msg):
            hq.attention(b, bad, buf, buf, 1.0)
    for kw, msg in ((dict(q_stride=4), "strides"), (dict(out_stride=64), "strides"), (dict(gate=buf.ptr + 2), "aligned to 4"),
                    (dict(gate=buf.ptr, gate_stride=2), "gate strides")):
        with pytest.raises(hq.HQError, match=msg):
            hq.attention(b, kv, buf, buf, 1.0, **kw)
    for a, msg in (((buf.ptr + 2, buf, 1.0), "16-byte"), ((None, buf, 1.0), "null"), ((buf, buf, float("nan")), "scale")):
        with pytest.raises(hq.HQError, match=msg):
            hq.attention(b, kv, *a)
    rope = dict(f32=True, q_stride=256, kv_stride=256)
    for kw, msg in ((dict(q_stride=4), "strides"), (dict(q_head_stride=32), "strides"), (dict(q_norm=buf), "q_norm without"),
                    (dict(positions=buf), "axes"), (dict(positions=buf, axis=np.full(32, 8, np.uint8)), "axes")):
        with pytest.raises(hq.HQError, match=msg):
            hq.rope_append(b, kv, buf, buf, buf, buf, buf, 16, 64, **dict(rope, **kw))
    for rot, n, msg in ((12, 16, "rot_dim"), (72, 16, "rot_dim"), (64, 0, "table")):
        with pytest.raises(hq.HQError, match=msg):
            hq.rope_append(b, kv, buf, buf, buf, buf, buf, n, rot, **rope)
    with pytest.raises(hq.HQError, match="inv_freq|rot_dim"):
        hq.rope_table(np.ones(129, np.float32), 4, buf)
    # a step without tokens is no error, and queues nothing
    b.set(kv, 2, [0, 0], [1, 0], np.array([[0], [0]]))
    hq.attention(b, kv, None, None, 1.0)
    b.set(kv, 2, [], [], np.zeros((0, 1)))
    hq.attention(b, kv, None, None, 1.0)
    b.free()
