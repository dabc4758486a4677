"""hq_delta with its norm and gate: outputs of any size before the norm, by chunks as token by token, rounded to fp16 once.

Bounds: delta_ref's of the outputs before the norm, without their rounding to fp16 (which its form with a norm has), through the norm's
formula. They are worst cases of sums that cancel; what a further rounding does shows in the root mean square: errors r of the one
rounding to fp16 (formed of the float64 values) and independent ones of size e beside it have sqrt(r^2 + e^2), and 1.1 r leaves e 0.46 r, some
2^-14 of the outputs, where states of 32 bits and operands of 22 have 2^-19. A second rounding to fp16 would make it 1.4 r."""
import numpy as np
import pytest

from delta_ref import U16, U32, delta, silu
from test_gpu_delta import go, inputs, split

pytestmark = pytest.mark.gpu


def normed(o, b, gate, norm, eps):
    """The outputs behind norm and gate of outputs o [tokens, heads, dv] that are off by b, and their bound."""
    z = silu(gate.astype(np.float64)) * norm.astype(np.float64)
    ms = (o * o).mean(-1, keepdims=True) + eps
    rel = (np.abs(o) * b).mean(-1, keepdims=True) / ms + (o.shape[-1] + 16) * U32
    y = o / np.sqrt(ms) * z
    return y, (b + np.abs(o) * rel) / np.sqrt(ms) * np.abs(z) * (1 + 2 * rel) + U16 * np.abs(y) + 2.0 ** -25


def check(hqlib, seed, hk, hv, dk, dv, seqs, size, eps, gate_type=np.float32, by="scale"):
    """Outputs of a root mean square of about `size` before the norm."""
    rng = np.random.default_rng(seed)
    n_new, src, dst = [list(a) for a in zip(*seqs)]
    x, g, beta = inputs(rng, sum(n_new), hk, hv, dk, dv)
    states = rng.normal(0, 0.5, (max(src + dst) + 2, hv, dk, dv)).astype(np.float32)
    scale = 1.0
    before = [states[i] if i >= 0 else np.zeros((hv, dk, dv), np.float32) for i in src]
    o, *_ = delta(*split(x, hk, hv, dk, dv), g, beta, before, n_new, 1.0)
    factor = size / np.sqrt((o * o).mean())
    if by == "scale":
        scale = float(np.float32(factor))
    else:
        states *= np.float32(factor)
        x[:, 2 * hk * dk:] = (x[:, 2 * hk * dk:].astype(np.float64) * factor).astype(np.float16)
        before = [states[i] if i >= 0 else np.zeros((hv, dk, dv), np.float32) for i in src]
    gate, norm = rng.normal(0, 2, (sum(n_new), hv, dv)).astype(gate_type), rng.normal(1, 0.2, dv).astype(np.float32)
    print(f"[gpu] delta norm {hk}/{hv} x {dk}, {dv} {seqs} outputs of {size} by {by} eps={eps} {np.dtype(gate_type).name}", flush=True)
    y, s = go(hqlib, x, g, beta, states, n_new, src, dst, hk, hv, dk, dv, gate, norm, eps=eps, scale=scale)
    o, b, after, e = delta(*split(x, hk, hv, dk, dv), g, beta, before, n_new, scale)
    want, bound = normed(o, b - U16 * np.abs(o) - 2.0 ** -25, gate, norm, eps)
    assert np.isfinite(y).all()
    assert (np.abs(y - want) <= bound).all(), np.max(np.abs(y - want) / bound)
    once = np.sqrt(((want.astype(np.float16).astype(np.float64) - want) ** 2).mean())
    assert np.sqrt(((y - want) ** 2).mean()) <= 1.1 * once
    for i, a, d in zip(dst, after, e):
        if i >= 0:
            assert (np.abs(s[i] - a) <= d).all()


STEPS, CHUNKS, BOTH = [(8, 0, 0), (3, -1, 1)], [(130, 0, 1), (64, -1, 2), (65, 3, 3)], [(200, 0, 0), (3, 1, 1), (17, -1, 2)]


@pytest.mark.parametrize("seqs", [STEPS, CHUNKS, BOTH], ids=["tokens", "chunks", "both"])
@pytest.mark.parametrize("size,eps", [(1e-6, 1e-6), (1e-5, 1e-6), (1e-3, 1e-6), (1.0, 1e-6), (1e5, 1e-6), (1e9, 1e-6), (1e-6, 0.0), (1e-9, 1e-18)])
def test_sizes_by_scale(hqlib, seqs, size, eps):
    check(hqlib, 1, 1, 2, 128, 128, seqs, size, eps)


@pytest.mark.parametrize("seqs", [STEPS, CHUNKS], ids=["tokens", "chunks"])
@pytest.mark.parametrize("size", [1e-2, 1e2])
def test_sizes_by_values(hqlib, seqs, size):
    """Values and states that make the outputs small or large themselves."""
    check(hqlib, 2, 1, 2, 128, 128, seqs, size, 1e-6, np.float16, by="values")


@pytest.mark.parametrize("hk,hv,dk,dv,seqs", [
    (1, 1, 16, 16, [(130, 0, 0)]), (1, 2, 64, 64, [(300, 0, 1), (1, 2, 2)]), (1, 1, 96, 192, [(129, -1, 0)]), (1, 1, 256, 256, [(70, 0, 0)]), (2, 2, 48, 80, [(100, 0, 0)]),
    (1, 1, 256, 32, [(66, 0, 0)]), (1, 2, 128, 128, [(1601, 0, 1)]), (1, 1, 48, 256, [(1217, 0, 0)])])
@pytest.mark.parametrize("size", [1e-6, 1e6])
def test_shapes(hqlib, hk, hv, dk, dv, seqs, size):
    """Other heads, parts of a sequence, rows of the workspace that the heads do not fill."""
    check(hqlib, 3 + dk, hk, hv, dk, dv, seqs, size, 1e-9, [np.float16, np.float32][dk % 3 % 2])


def test_the_company_of_other_sequences(hqlib):
    """A sequence's outputs, large before the norm, agree within their bounds and stay finite whether it goes token by token or by chunks,
    which the step's other sequences decide."""
    hk, hv, dk, dv, n = 1, 2, 64, 64, 12
    rng = np.random.default_rng(4)
    x, g, beta = inputs(rng, n + 400, hk, hv, dk, dv)
    states = (1e5 * rng.normal(0, 0.5, (3, hv, dk, dv))).astype(np.float32)
    gate, norm = rng.normal(0, 2, (n + 400, hv, dv)).astype(np.float32), rng.normal(1, 0.2, dv).astype(np.float32)
    o, b, *_ = delta(*split(x[:n], hk, hv, dk, dv), g[:n], beta[:n], [states[0]], [n], 10.0)
    want, bound = normed(o, b - U16 * np.abs(o) - 2.0 ** -25, gate[:n], norm, 1e-6)
    assert np.abs(o).max() > 1e6
    for parts in ([n], [n, 400], [n] + [1] * 200, [6, 6]):
        print(f"[gpu] delta norm {parts[:3]} of {len(parts)}", flush=True)
        T = sum(parts)
        if parts == [6, 6]:  # its tokens by two steps, token by token
            y, s = go(hqlib, x[:6], g[:6], beta[:6], states, [6], [0], [0], hk, hv, dk, dv, gate[:6], norm, eps=1e-6, scale=10.0)
            z, _ = go(hqlib, x[6:n], g[6:n], beta[6:n], s, [6], [0], [0], hk, hv, dk, dv, gate[6:n], norm, eps=1e-6, scale=10.0)
            y = np.concatenate([y, z])
        else:
            m = len(parts)
            y, _ = go(hqlib, x[:T], g[:T], beta[:T], states, parts, [0] + [-1] * (m - 1), [-1] * m, hk, hv, dk, dv, gate[:T], norm, eps=1e-6, scale=10.0)
        assert (np.abs(y[:n] - want) <= bound).all(), parts[:3]


@pytest.mark.parametrize("seqs", [STEPS, CHUNKS], ids=["tokens", "chunks"])
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 32), (96, 192)])
@pytest.mark.parametrize("size,eps", [(4e18, 1e-6), (3e19, 0.0), (1e-16, 0.0), (1e-25, 0.0), (1e-30, 1e-38)])
def test_squares_beyond_fp32(hqlib, seqs, dk, dv, size, eps):
    """Outputs whose squares pass fp32's range, or vanish in it, through the scale that hq_delta takes."""
    hk, hv = 1, 2
    rng = np.random.default_rng(5)
    n_new, src, dst = [list(a) for a in zip(*seqs)]
    x, g, beta = inputs(rng, sum(n_new), hk, hv, dk, dv)
    x[1, 2 * hk * dk:] = 0
    beta[1] = 0
    states = rng.normal(0, 4, (max(src + dst) + 2, hv, dk, dv)).astype(np.float32)
    before = [states[i] if i >= 0 else np.zeros((hv, dk, dv), np.float32) for i in src]
    o, b, after, e = delta(*split(x, hk, hv, dk, dv), g, beta, before, n_new, 1.0)
    b = b - U16 * np.abs(o) - 2.0 ** -25
    scale = float(np.float32(min(size / np.sqrt((o * o).mean()), 1e20)))
    gate, norm = rng.normal(0, 2, (sum(n_new), hv, dv)).astype(np.float32), rng.normal(1, 0.2, dv).astype(np.float32)
    print(f"[gpu] delta norm {dk}, {dv} {seqs} outputs of {size} eps={eps}", flush=True)
    y, _ = go(hqlib, x, g, beta, states, n_new, src, dst, hk, hv, dk, dv, gate, norm, eps=eps, scale=scale)
    want, bound = normed(scale * o, scale * b, gate, norm, float(np.float32(eps)))
    assert (np.abs(y - want) <= bound).all()
    once = np.sqrt(((want.astype(np.float16).astype(np.float64) - want) ** 2).mean())
    assert np.sqrt(((y - want) ** 2).mean()) <= 1.1 * once


@pytest.mark.parametrize("seqs", [STEPS, CHUNKS], ids=["tokens", "chunks"])
def test_outputs_beyond_fp32(hqlib, seqs):
    """Outputs that the scale would take beyond fp32 (one column of 1e45 and more: it has the head's norm, and the others are nothing beside it);
    rows of zeros, which are 0 for eps above 0."""
    hk, hv, dk, dv = 1, 1, 64, 64
    rng = np.random.default_rng(6)
    n_new, src, dst = [list(a) for a in zip(*seqs)]
    T = sum(n_new)
    x, g, beta = inputs(rng, T, hk, hv, dk, dv)
    states = rng.normal(0, 4, (max(src + dst) + 2, hv, dk, dv)).astype(np.float32)
    x[2, :hk * dk] = 0  # a query of zeros
    states[0, 0, :, 5] = 1e30
    x[:, :2 * hk * dk] = np.abs(x[:, :2 * hk * dk])  # (queries and keys of one sign: nothing cancels in the column)
    g[:3], beta[:3] = 0, 0
    gate, norm = rng.normal(0, 2, (T, hv, dv)).astype(np.float32), np.ones(dv, np.float32)
    print(f"[gpu] delta norm beyond fp32 {seqs}", flush=True)
    y, _ = go(hqlib, x, g, beta, states, n_new, src, [-1] * len(dst), hk, hv, dk, dv, gate, norm, eps=1e-6, scale=1e15)
    before = [states[i] if i >= 0 else np.zeros((hv, dk, dv), np.float32) for i in src]
    o, b, *_ = delta(*split(x, hk, hv, dk, dv), g, beta, before, n_new, 1.0)
    want, bound = normed(1e15 * o, 1e15 * (b - U16 * np.abs(o) - 2.0 ** -25), gate, norm, 1e-6)
    assert (np.abs(want[:2, 0, 5] / silu(gate[:2, 0, 5].astype(np.float64)) - 8) < 1e-6).all() and (want[2] == 0).all()
    assert (np.abs(y[:3] - want[:3]) <= bound[:3]).all()
