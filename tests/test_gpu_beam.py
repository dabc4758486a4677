"""hq_beam against a float64 selection. Scores: a value is formed in 64 bits from a row's sum that is off by 2^-21 of itself at
most (its exponentials 2^-22, sums of eight of them 3 * 2^-24), so values are off by 2^-20, and the fp32 result by 2^-24 of itself
more. Choices: places may only differ from float64's where the values there are nearer than twice that; inputs are drawn so that
none is."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def choose(x, score, done, done_token, k):
    """x [groups, beams, V], score [groups, beams]: (score, token, beam) [groups, k] and how near a choice was."""
    G, B, V = x.shape
    out = np.full((G, k), -np.inf), np.full((G, k), 0xffffffff, np.uint32), np.full((G, k), -1, np.int32)
    gap = np.inf
    for i in range(G):
        val, tok, bm = [], [], []
        for b in range(B):
            if done is not None and done[i, b]:
                val.append([float(score[i, b])]), tok.append([done_token]), bm.append([b])
                continue
            row = x[i, b].astype(np.float64)
            with np.errstate(invalid="ignore", divide="ignore"):
                m = row.max()
                lp = row - m - np.log(np.exp(row - m).sum()) if np.isfinite(m) else np.full(V, -np.inf)
            top = np.lexsort((np.arange(V), -row))[:k + 1]
            val.append(float(score[i, b]) + lp[top]), tok.append(top), bm.append(np.full(len(top), b))
        val, tok, bm = (np.concatenate(a) for a in (val, tok, bm))
        at = np.lexsort((tok, bm, -val))
        at = at[val[at] > -np.inf][:k + 1]
        same = (val[at][1:] == val[at][:-1]) & (bm[at][1:] == bm[at][:-1])  # ties within a row are exact
        d = np.where(same, np.inf, val[at][:-1] - val[at][1:])
        gap = min(gap, d.min(initial=np.inf))
        at = at[:k]
        out[0][i, :len(at)], out[1][i, :len(at)], out[2][i, :len(at)] = val[at], tok[at], bm[at]
    return out, gap


def go(hqlib, x, score, k, done=None, done_token=0, pad=0, stream=None, check=True):
    G, B, V = x.shape
    rows = np.full((G * B, V + pad), np.nan, x.dtype)
    rows[:, :V] = x.reshape(G * B, V)
    d = [hqlib.DevBuf.from_array(a) for a in (rows, score.astype(np.float32))] + [None if done is None else hqlib.DevBuf.from_array(done.astype(np.uint8))]
    out = [hqlib.DevBuf.from_array(np.full(G * k + 1, 77, np.uint32)) for _ in range(3)]
    hqlib.beam(d[0], G, B, V, d[1], k, *out, f32=x.dtype == np.float32, stride=V + pad, done=d[2], done_token=done_token, stream=stream)
    hqlib.synchronize()
    got = [o.download(G * k + 1, t) for o, t in zip(out, (np.float32, np.uint32, np.int32))]
    assert all(g.view(np.uint32)[-1] == 77 for g in got)
    got = [g[:-1].reshape(G, k) for g in got]
    if check:
        want, gap = choose(x, score.astype(np.float32), done, done_token, k)
        assert gap > 2.0 ** -19, "the inputs leave a choice open"
        assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
        fin = np.isfinite(want[0])
        assert np.array_equal(np.isfinite(got[0]), fin) and (got[0][~fin] == -np.inf).all()
        assert (np.abs(got[0] - want[0])[fin] <= 2.0 ** -20 + 2.0 ** -24 * np.abs(want[0][fin])).all()
    return got


def draw(rng, G, B, V, f32, std=3.0):
    """Logits whose candidates lie apart: multiples of 2^-6 a row, scores that keep the rows' values off each other."""
    x = (np.rint(rng.normal(0, std, (G, B, V)) * 64) / 64).astype(np.float32 if f32 else np.float16)
    return x, rng.uniform(-20, 0, (G, B)).astype(np.float32)


CASES = [  # groups, beams, V, k, f32, values of other use behind a row
    (1, 1, 1, 1, True, 0), (1, 1, 5, 5, True, 3), (3, 2, 7, 16, False, 1), (1, 4, 32000, 8, True, 0), (5, 3, 1000, 7, False, 5), (2, 16, 151936, 32, True, 0),
    (16, 8, 20011, 16, False, 2), (1, 64, 4099, 64, True, 1), (600, 1, 513, 2, True, 0), (100, 5, 3001, 10, False, 0), (4, 64, 100, 64, False, 0), (1, 2, 300001, 64, True, 3)]


@pytest.mark.parametrize("G,B,V,k,f32,pad", CASES)
def test_beam(hqlib, G, B, V, k, f32, pad):
    print(f"[gpu] beam {G} x {B} of {V} k {k} f32={f32}", flush=True)
    x, score = draw(np.random.default_rng(G + B + V), G, B, V, f32)
    a = go(hqlib, x, score, k, pad=pad)
    assert all(np.array_equal(p, q) for p, q in zip(a, go(hqlib, x, score, k, pad=pad)))  # workspaces are left as they were found


def test_masks_ends_and_first_steps(hqlib):
    rng = np.random.default_rng(11)
    G, B, V, k = 9, 6, 4001, 12
    x, score = draw(rng, G, B, V, True)
    x[rng.random(x.shape) < 0.4] = -np.inf
    done = rng.random((G, B)) < 0.3
    x[0, 1] = -np.inf           # nothing is allowed
    x[0, 2, 1:] = -np.inf       # one token is
    score[1, 1:] = -np.inf      # a request's first step
    done[1, 1:3] = True         # (ended and worth nothing: no candidate)
    done[1, 0] = False
    score[2], done[2] = -np.inf, False  # no candidates at all
    done[3] = True              # six candidates for twelve places
    x[4, done[4]] = np.nan      # rows that nobody reads
    x[1, 1:] = np.nan
    x[2] = np.inf
    got = go(hqlib, x, score, k, done, 17)
    assert (got[2][2] == -1).all() and (got[1][2] == 0xffffffff).all() and (got[2][3, 6:] == -1).all() and (got[1][3, :6] == 17).all()


def test_without_a_number(hqlib):
    """A NaN or +inf in a row or a score that counts: the group has no choice, the others keep theirs."""
    rng = np.random.default_rng(12)
    G, B, V, k = 6, 3, 30011, 5
    x, score = draw(rng, G, B, V, True)
    want = go(hqlib, x, score, k)
    x[0, 1, 30010], x[1, 2, 0], score[2, 0], score[3, 2] = np.nan, np.inf, np.nan, np.inf
    got = go(hqlib, x, score, k, check=False)
    assert np.isnan(got[0][:4]).all() and (got[1][:4] == 0xffffffff).all() and (got[2][:4] == -1).all()
    assert all(np.array_equal(a[4:], b[4:]) for a, b in zip(got, want))


def test_ties(hqlib):
    """Equal values: the lower beam, then the lower token; more equal logits than places; rows in falling and rising order."""
    V, k = 5000, 8
    x = np.zeros((1, 3, V), np.float32)
    got = go(hqlib, x, np.array([[-1, -1, -1]]), k, check=False)
    assert got[1].tolist() == [list(range(8))] and got[2].tolist() == [[0] * 8] and len(set(got[0][0])) == 1
    x[0, :, 100::7] = 2
    x[0, 1] = x[0, 1, ::-1]
    got = go(hqlib, x, np.array([[-5, -1, -1.5]]), 64)
    assert (got[2] == 1).all() and np.array_equal(got[1][0], np.flatnonzero(x[0, 1] == 2)[:64])
    x = np.stack([np.arange(V), np.arange(V)[::-1]]).astype(np.float32)[None] * np.float32(2.0 ** -5)
    go(hqlib, x, np.array([[-1, -1.01]]), 32)


def test_large_scores(hqlib):
    """Rows whose logits are large as a whole, and sums of a long search."""
    rng = np.random.default_rng(13)
    x, score = draw(rng, 4, 4, 9001, True)
    x[0] += 3e4
    x[1] -= 1e6
    score[2] -= 300
    go(hqlib, x, score, 8)


def test_two_streams(hqlib):
    rng = np.random.default_rng(14)
    s = [hqlib.Stream(), hqlib.Stream()]
    for G, V in ((1, 90000), (40, 3000), (2, 200)):
        for st in s:
            go(hqlib, *draw(rng, G, 4, V, True), 8, stream=st.ptr)
    for st in s:
        st.destroy()


@pytest.mark.parametrize("G,B,V,k", [(1, 4, 3000, 8), (20, 3, 17000, 6)])
def test_lowest_values(hqlib, G, B, V, k):
    """fp32 rows barred with the type's lowest value, rows of nothing else (all tokens alike), and logits near either end of the type."""
    print(f"[gpu] beam lowest values {G} x {B} of {V}", flush=True)
    lowest = np.finfo(np.float32).min
    x, score = draw(np.random.default_rng(V), G, B, V, True)
    x[np.random.default_rng(V + 1).random(x.shape) < 0.7] = lowest
    x[0, 1] = lowest                      # every token 1 / V
    x[0, 2] = -np.inf
    x[0, 2, ::3], score[0, 2] = lowest, -25  # every third token, and worth less than row 1's
    score[0, 1] = -0.25
    if G > 1:
        x[1, 0, 5], x[1, 0, 6] = 3e38, 2.9e38  # one token has it all
        x[2, 1, :] = np.where(np.arange(V) < V // 2, np.float32(-2.0 ** 100), np.float32(-2.0 ** 100 * (1 - 2.0 ** -24)))
        score[2] = -30, -1, -40
    go(hqlib, x, score, k)
    y = np.full((1, 2, V), lowest, np.float32)
    y[0, 1] = -np.inf
    got = go(hqlib, y, np.array([[-0.5, -0.1]]), k)
    assert got[1].tolist() == [list(range(k))] and (got[2] == 0).all() and np.allclose(got[0], -0.5 - np.log(V), rtol=0, atol=2.0 ** -20)


def test_more_places_than_a_row_has(hqlib):
    """Rows shorter than k: places come from several beams, and their number need not be a power of two."""
    for B, V, k in ((3, 4, 11), (5, 2, 10), (64, 1, 64), (7, 9, 64)):
        x, score = draw(np.random.default_rng(B), 2, B, V, True)
        x += np.linspace(0, 2.0 ** -8, x.size, dtype=np.float32).reshape(x.shape)  # (no two alike)
        go(hqlib, x, score, k)


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("at", [0.0, 60000.0, -60000.0, 131071.0, 131073.0, -131073.0, 1.5e6, -2.0e30])
def test_where_logits_lie(hqlib, f32, at):
    """Rows whose largest logits lie anywhere: near 0, at fp16's ends, and on both sides of 2^17, thread by thread."""
    if not f32 and abs(at) > 65504:
        at = np.sign(at) * 65000.0
    rng = np.random.default_rng(int(abs(at) % 1000))
    G, B, V, k = 2, 3, 40000, 4
    x = (at + rng.integers(-64, 1, (G, B, V)) / 8.0).astype(np.float32 if f32 else np.float16)
    x[:, 1, rng.random(V) < 0.5] = -6e4
    go(hqlib, x, rng.uniform(-20, 0, (G, B)).astype(np.float32), k)
