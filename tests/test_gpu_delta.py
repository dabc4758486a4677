"""hq_delta against a float64 recurrence (tests/delta_ref.py, where the bounds are derived)."""
import numpy as np
import pytest

from delta_ref import delta

pytestmark = pytest.mark.gpu


def inputs(rng, T, hk, hv, dk, dv, pad=8):
    """q | k | v rows with `pad` values of other use at the end, keys and queries of norm 1 and alike (as behind a SiLU), decays from
    near 1 to near 0, write strengths over 0 .. 1."""
    x = rng.normal(0.5, 1, (T, 2 * hk * dk + hv * dv + pad))
    n = x[:, :2 * hk * dk].reshape(T, 2 * hk, dk)
    n /= np.linalg.norm(n, axis=-1, keepdims=True) * 1.001  # (fp16 may round up: norms stay below 1)
    g = -np.exp(rng.uniform(-7, 2, (T, hv)))
    return x.astype(np.float16), g.astype(np.float32), rng.uniform(0, 1, (T, hv)).astype(np.float32)


def split(x, hk, hv, dk, dv):
    T, c = x.shape[0], hk * dk
    return x[:, :c].reshape(T, hk, dk), x[:, c:2 * c].reshape(T, hk, dk), x[:, 2 * c:2 * c + hv * dv].reshape(T, hv, dv)


def go(hqlib, x, g, beta, states, n_new, src, dst, hk, hv, dk, dv, gate=None, norm=None, eps=1e-5, scale=None, stream=None, scan=None):
    """hq_delta with gaps in its strides; outputs and states, after checks that nothing else was written."""
    T, slots = x.shape[0], states.shape[0]
    scale = dk ** -0.5 if scale is None else scale
    d = [hqlib.DevBuf.from_array(a) for a in (x if T else np.zeros(8, np.float16), g if T else np.zeros(8, np.float32), beta if T else np.zeros(8, np.float32), states)]
    st = hqlib.States(hk, hv, dk, dv, 1, slots, d[3], None)
    own = scan is None
    scan = hqlib.Scan(len(n_new), T) if own else scan
    scan.set(st, n_new, src, dst, stream=stream)
    ld = hv * dv + 16
    out = hqlib.DevBuf.from_array(np.full((T + 1, ld), 7, np.float16))
    kw = {}
    if gate is not None:
        z = np.full((T + 1, ld), np.nan, gate.dtype)
        z[:T, :hv * dv] = gate.reshape(T, -1)
        d += [hqlib.DevBuf.from_array(z), hqlib.DevBuf.from_array(norm)]
        kw = dict(norm=d[5], gate=d[4], gate_f32=gate.dtype == np.float32, gate_stride=ld, eps=eps)
    hqlib.delta(scan, st, d[0], d[0].ptr + 2 * hk * dk, d[0].ptr + 4 * hk * dk, d[1], d[2], out, scale, qk_stride=x.shape[1], v_stride=x.shape[1],
                out_stride=ld, stream=stream, **kw)
    hqlib.synchronize()
    y = out.download((T + 1, ld), np.float16)
    assert (y[T] == 7).all() and (y[:, hv * dv:] == 7).all()
    s = d[3].download(states.shape, np.float32)
    kept = [i for i in range(slots) if i not in dst]
    assert np.array_equal(s[kept].view(np.uint32), states[kept].view(np.uint32))
    if own:
        scan.free()
    return y[:T, :hv * dv].reshape(T, hv, dv).astype(np.float64), s


def check(hqlib, seed, hk, hv, dk, dv, seqs, gate_type=None, change=None, **kw):
    rng = np.random.default_rng(seed)
    n_new, src, dst = [list(a) for a in zip(*seqs)]
    T, slots = sum(n_new), max(src + dst) + 2
    x, g, beta = inputs(rng, T, hk, hv, dk, dv)
    states = np.full((slots, hv, dk, dv), np.nan, np.float32)
    for s in src:
        if s >= 0:
            states[s] = rng.normal(0, 0.5, (hv, dk, dv))
    if change:
        change(x, g, beta, states)
    gate = norm = None
    if gate_type:
        gate, norm = rng.normal(0, 2, (T, hv, dv)).astype(gate_type), rng.normal(1, 0.2, dv).astype(np.float32)
    print(f"[gpu] delta {hk}/{hv} x {dk}, {dv} {seqs} gate={gate_type}", flush=True)
    y, s = go(hqlib, x, g, beta, states, n_new, src, dst, hk, hv, dk, dv, gate, norm, **kw)
    before = [states[i] if i >= 0 else np.zeros((hv, dk, dv), np.float32) for i in src]
    want, bound, after, e = delta(*split(x, hk, hv, dk, dv), g, beta, before, n_new, kw.get("scale") or dk ** -0.5, norm, gate, kw.get("eps", 1e-5))
    assert (np.abs(y - want) <= bound).all(), np.max(np.abs(y - want) / bound)
    for i, a, b in zip(dst, after, e):
        if i >= 0:
            assert (np.abs(s[i] - a) <= b + U_MIN).all()
            # errors are random: far below the sum of their bounds
            size = np.sqrt((a * a).mean())
            assert np.sqrt(((s[i] - a) ** 2).mean()) <= 2.0 ** -19 * size + U_MIN
    return y, s


U_MIN = 2.0 ** -126

CASES = [  # key heads, value heads, k_dim, v_dim, (new, from, to) of each sequence, gate
    (1, 1, 16, 16, [(1, -1, 0)], None),
    (1, 1, 128, 128, [(1, 0, 0)], np.float16),
    (2, 4, 64, 64, [(1, 0, 3), (2, -1, 1), (0, 2, 4), (5, 2, 2 + 3)], np.float32),
    (1, 2, 128, 128, [(63, 0, 0), (64, -1, 1), (65, 2, 3), (1, 4, 4), (0, -1, 5), (0, 2, 6), (17, 2, -1)], None),
    (1, 2, 128, 128, [(200, 0, 0), (16, 1, 1), (9, -1, 2)], np.float16),
    (1, 1, 96, 192, [(130, -1, 0), (3, 1, 1)], np.float32),
    (1, 1, 48, 80, [(70, 0, 0), (31, -1, 1)], np.float16),
    (1, 3, 16, 256, [(33, -1, 0), (128, 1, 1)], None),
    (1, 1, 256, 256, [(129, 0, 1), (7, -1, 2)], np.float32),
    (1, 1, 256, 32, [(66, 0, 0)], None),
    (2, 2, 112, 48, [(20, -1, 0), (100, 1, 1)], None),
    (16, 32, 128, 128, [(1, 0, 0), (12, 1, 1)], np.float32),
    (1, 1, 32, 64, [(700, -1, 0)], None),
]


@pytest.mark.parametrize("hk,hv,dk,dv,seqs,gate", CASES)
def test_delta(hqlib, hk, hv, dk, dv, seqs, gate):
    check(hqlib, dk + dv + hv, hk, hv, dk, dv, seqs, gate)


LENS = [(130, 0, 0), (1, 1, 1), (5, -1, 2)]


def test_edges_of_gates(hqlib):
    """Decays of nothing (-inf), of everything kept (0) and far below any fp32 exponential; write strengths of 0 and 1; keys and
    queries of zeros."""
    def change(x, g, beta, states):
        g[::7] = -np.inf
        g[1::7] = 0
        g[2::7] = -1e4
        g[64:70] = -np.inf
        beta[::5], beta[1::5] = 0, 1
        x[3::11, :256] = 0
    check(hqlib, 3, 1, 2, 128, 128, LENS, change=change)


def test_same_key_again(hqlib):
    """One key all along, written with full strength and never decayed: the state holds the last value."""
    def change(x, g, beta, states):
        x[:, 128:256] = x[0, 128:256]
        g[:], beta[:] = 0, 1
    check(hqlib, 4, 1, 1, 128, 64, LENS, change=change)


@pytest.mark.parametrize("size", [2.0 ** -12, 1e4])
def test_sizes_of_values(hqlib, size):
    """Values and states that are small or large as a whole, and of unlike size in neighbouring columns."""
    def change(x, g, beta, states):
        x[:, 256:384] = (x[:, 256:384].astype(np.float32) * size * np.where(np.arange(128) % 2, 1, 2.0 ** -6)).astype(np.float16)
        states *= np.float32(size)
        states[..., ::2] *= 2.0 ** 10
    check(hqlib, 5, 1, 1, 128, 128, LENS, change=change, scale=1.0 / size)


def test_a_bad_value_stays_in_its_place(hqlib):
    """A NaN in one value column makes that column NaN from its token on, and no other column, head or sequence."""
    rng = np.random.default_rng(6)
    n_new, src, dst, hk, hv, dk, dv = [100, 40], [0, 1], [0, 1], 1, 2, 64, 64
    x, g, beta = inputs(rng, 140, hk, hv, dk, dv)
    states = rng.normal(0, 0.5, (3, hv, dk, dv)).astype(np.float32)
    want, s_want = go(hqlib, x, g, beta, states, n_new, src, dst, hk, hv, dk, dv)
    x[70, 2 * hk * dk + dv + 5] = np.nan  # head 1, column 5
    y, s = go(hqlib, x, g, beta, states, n_new, src, dst, hk, hv, dk, dv)
    assert np.isnan(y[70:100, 1, 5]).all() and np.isnan(s[0, 1, :, 5]).all()
    y[64:100, 1, 5], s[0, 1, :, 5] = want[64:100, 1, 5], s_want[0, 1, :, 5]  # (tokens of the same chunk before it may be NaN too)
    assert np.array_equal(y, want) and np.array_equal(s, s_want)


def test_same_bits_and_any_split(hqlib):
    """The same step gives the same bits; a prompt in pieces agrees with the whole within the bound."""
    hk, hv, dk, dv, n = 1, 2, 128, 128, 300
    rng = np.random.default_rng(7)
    x, g, beta = inputs(rng, n, hk, hv, dk, dv)
    states = rng.normal(0, 0.5, (2, hv, dk, dv)).astype(np.float32)
    a = go(hqlib, x, g, beta, states, [n], [0], [1], hk, hv, dk, dv)
    b = go(hqlib, x, g, beta, states, [n], [0], [1], hk, hv, dk, dv)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    want, bound, after, e = delta(*split(x, hk, hv, dk, dv), g, beta, [states[0]], [n], dk ** -0.5)
    at, s, y = 0, states, []
    for m in (1, 64, 130, 7, 98):
        r = slice(at, at + m)
        o, s = go(hqlib, x[r], g[r], beta[r], s, [m], [0], [0], hk, hv, dk, dv)
        y.append(o)
        at += m
    assert (np.abs(np.concatenate(y) - want) <= bound).all() and (np.abs(s[0] - after[0]) <= e[0]).all()


def test_branches(hqlib):
    """Three sequences go on from one slot with tokens of their own, as three copies of the state would."""
    hk, hv, dk, dv = 1, 2, 64, 64
    rng = np.random.default_rng(8)
    x, g, beta = inputs(rng, 75, hk, hv, dk, dv)
    states = rng.normal(0, 0.5, (4, hv, dk, dv)).astype(np.float32)
    states[1:] = states[0]
    a = go(hqlib, x, g, beta, states, [5, 1, 69], [0, 0, 0], [1, 2, 3], hk, hv, dk, dv)
    b = go(hqlib, x, g, beta, states, [5, 1, 69], [1, 2, 3], [1, 2, 3], hk, hv, dk, dv)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_two_steps_on_two_streams(hqlib):
    """Steps that overlap in time, each with a Scan of its own; one Scan set again and again."""
    hk, hv, dk, dv = 1, 2, 128, 128
    rng = np.random.default_rng(9)
    streams = [hqlib.Stream(), hqlib.Stream()]
    scans = [hqlib.Scan(4, 400), hqlib.Scan(4, 400)]
    for n_new in ([300, 1], [1, 1, 1], [20, 70, 0, 2], [1]):
        for i in range(2):
            n = len(n_new)
            x, g, beta = inputs(rng, sum(n_new), hk, hv, dk, dv)
            states = rng.normal(0, 0.5, (n + 1, hv, dk, dv)).astype(np.float32)
            y, s = go(hqlib, x, g, beta, states, n_new, list(range(n)), list(range(n)), hk, hv, dk, dv, stream=streams[i].ptr, scan=scans[i])
            want, bound, after, e = delta(*split(x, hk, hv, dk, dv), g, beta, states[:n], n_new, dk ** -0.5)
            assert (np.abs(y - want) <= bound).all()
            assert all((np.abs(s[j] - after[j]) <= e[j]).all() for j in range(n))
    for s in scans:
        s.free()
    for s in streams:
        s.destroy()


def test_refusals(hqlib):
    D = hqlib.DevBuf
    st = hqlib.States(1, 2, 64, 64, 4, 4, D(4 * 2 * 64 * 64 * 4), None)
    scan, x = hqlib.Scan(2, 8), D(64 * 1024)
    ok = dict(scan=scan, states=st, q=x, k=x, v=x, decay=x, beta=x, out=x, scale=1.0, qk_stride=256, v_stride=256)
    with pytest.raises(hqlib.HQError, match="no step"):
        hqlib.delta(**ok)
    scan.set(st, [1, 2], [-1, 3], [0, 1])
    for kw, text in ((dict(q=x.ptr + 8), "16-byte"), (dict(v=None), "null"), (dict(out=x.ptr + 4), "16-byte"), (dict(qk_stride=260), "stride 260"), (dict(v_stride=-8), "stride -8"),
                     (dict(out_stride=4), "stride 4"), (dict(norm=x), "without gate"), (dict(gate=x), "without gate"), (dict(norm=x, gate=x, gate_stride=12), "stride 12"),
                     (dict(norm=x, gate=x.ptr + 8), "16-byte"), (dict(norm=x, gate=x, eps=-1.0), "eps"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
                     (dict(decay=x.ptr + 2), "misaligned"), (dict(states=hqlib.States(1, 2, 64, 64, 4, 4, None, None)), "memory of the states"),
                     (dict(states=hqlib.States(2, 2, 64, 64, 4, 4, x, None)), "not those")):
        with pytest.raises(hqlib.HQError, match=text):
            hqlib.delta(**{**ok, **kw})
    scan.free()


@pytest.mark.parametrize("hk,hv,dk,dv,seqs,gate", [
    (2, 2, 64, 64, [(1500, 0, 0)], None),                                   # one long sequence, its state in its place
    (1, 2, 128, 128, [(1601, 1, 3)], np.float32),
    (1, 1, 128, 32, [(1000, -1, -1), (900, -1, 0), (40, 1, 1), (3, 2, 2)], np.float16),  # beginnings, nothing kept, short ones beside it
    (1, 2, 32, 128, [(1100, 0, 0), (0, 1, 2), (1025, 3, 4)], None),
    (1, 1, 256, 48, [(900, 0, 1)], None), (1, 1, 48, 256, [(1217, 0, 0)], np.float32),
    (3, 3, 16, 16, [(2100, -1, 0), (17, 2, 2)], None)])
def test_long_sequences_in_parts(hqlib, hk, hv, dk, dv, seqs, gate):
    """Few heads and long sequences: parts of a sequence side by side, with the states between them formed of their effects."""
    check(hqlib, 40 + hv + dk + dv, hk, hv, dk, dv, seqs, gate)


def test_parts_keep_what_is_not_a_number_apart(hqlib):
    """A value that is not a number, in the first part's state and in a middle part's values, stays in its column through the parts."""
    hk, hv, dk, dv, n = 1, 1, 64, 64, 1200
    rng = np.random.default_rng(9)
    x, g, beta = inputs(rng, n, hk, hv, dk, dv)
    states = np.zeros((2, hv, dk, dv), np.float32)
    states[0] = rng.normal(0, 0.5, (hv, dk, dv))
    print("[gpu] delta parts with NaN", flush=True)
    want, sw = go(hqlib, x, g, beta, states, [n], [0], [1], hk, hv, dk, dv)
    x[500, 2 * hk * dk + 7] = np.nan
    states[0, 0, 3, 50] = np.inf
    got, sg = go(hqlib, x, g, beta, states, [n], [0], [1], hk, hv, dk, dv)
    fine = [i for i in range(dv) if i not in (7, 50)]
    assert np.array_equal(got[:, :, fine], want[:, :, fine]) and np.array_equal(sg[1][:, :, fine], sw[1][:, :, fine])
    assert np.isnan(got[563:, 0, 7]).all() and np.isnan(got[63:, 0, 50]).all() and np.isnan(sg[1][0][:, [7, 50]]).all()
    assert np.array_equal(got[:448, 0, 7], want[:448, 0, 7])


@pytest.mark.parametrize("hk,hv,d,seqs,heads", [
    (64, 512, 16, [(300, 0, 0), (4500, 1, 2), (100, -1, 3)], (0, 8, 504)),  # 68 chunks of 512 heads to a pass of the workspace
    (8, 64, 16, [(36000, 0, 0)], (0,))])                                     # 538 of 64, and parts within each
def test_more_chunks_than_a_pass_has(hqlib, hk, hv, d, seqs, heads):
    """A sequence whose chunks do not fit the workspace together: its state goes on from pass to pass. (Heads are independent of each
    other: some of them are compared, two of one key head each.)"""
    n_new, src, dst = [list(a) for a in zip(*seqs)]
    rng = np.random.default_rng(hv)
    x, g, beta = inputs(rng, sum(n_new), hk, hv, d, d)
    states = rng.normal(0, 0.5, (max(dst) + 2, hv, d, d)).astype(np.float32)
    print(f"[gpu] delta passes {hk}/{hv} x {d} {seqs}", flush=True)
    y, s = go(hqlib, x, g, beta, states, n_new, src, dst, hk, hv, d, d)
    q, k, v = split(x, hk, hv, d, d)
    for h in heads:
        two, kh = slice(h, h + 2), slice(h // (hv // hk), h // (hv // hk) + 1)
        before = [states[i][two] if i >= 0 else np.zeros((2, d, d), np.float32) for i in src]
        want, bound, after, e = delta(q[:, kh], k[:, kh], v[:, two], g[:, two], beta[:, two], before, n_new, d ** -0.5)
        assert (np.abs(y[:, two] - want) <= bound).all()
        for i, a, b in zip(dst, after, e):
            assert (np.abs(s[i][two] - a) <= b + U_MIN).all() and np.sqrt(((s[i][two] - a) ** 2).mean()) <= 2.0 ** -19 * np.sqrt((a * a).mean())


@pytest.mark.parametrize("hk,hv,dk,dv,gate", [(4, 64, 64, 32, np.float32), (32, 64, 128, 64, None), (8, 72, 256, 48, np.float16), (5, 65, 48, 16, None)])
def test_some_tokens_of_many_heads(hqlib, hk, hv, dk, dv, gate):
    """Enough heads for sequences of up to 16 tokens to go token by token, eight at a time."""
    check(hqlib, 60 + hv, hk, hv, dk, dv, [(16, 0, 0), (9, 1, 6), (0, 2, 2), (1, -1, 3), (13, 3 + 1, -1), (8, 5, 7)], gate)


def test_some_tokens_of_few_heads(hqlib):
    """The same by chunks, a sequence of one token among them."""
    check(hqlib, 61, 1, 2, 128, 128, [(16, 0, 0), (9, 1, 6), (0, 2, 2), (1, -1, 3), (13, 3 + 1, -1), (8, 5, 7)], np.float32)
