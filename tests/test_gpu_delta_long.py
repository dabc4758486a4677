"""hq_delta over long sequences whose states last: what a part or a pass does to the state that it starts from counts in the result, as does the
bound of a column's unit over many chunks. (The draws of test_gpu_delta.inputs forget a state within a hundred tokens.)

In the root mean square states are within 2^-20 sqrt(chunks) of their size: each chunk's operands are two fp16 terms, off by 2^-22 of their column's
largest at most, which is some four times the mean, and errors of chunks are independent of each other. (A wrong matrix of a part is off by the
size of the state itself.) Every element is within delta_ref's bound besides."""
import os
import re

import numpy as np
import pytest

from delta_ref import delta
from test_gpu_delta import U_MIN, check, go, inputs, split

pytestmark = pytest.mark.gpu
CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "hilbert-pruned-8b_amd", "csrc")


def lasting(rng, T, hk, hv, dk, dv):
    """Decays of a ten thousandth to a hundredth a token, none at all in some heads, and small strengths."""
    x, g, beta = inputs(rng, T, hk, hv, dk, dv)
    g = -np.exp(rng.uniform(np.log(1e-4), np.log(1e-2), (T, hv))).astype(np.float32)
    g[:, ::3] /= 10
    g[:, 1::3] = 0
    return x, g, np.exp(rng.uniform(-8, -3, (T, hv))).astype(np.float32)


def compare(hqlib, seed, hk, hv, dk, dv, seqs, heads, part=256, draw=lasting):
    """Some value heads against the recurrence (heads are independent of each other)."""
    rng = np.random.default_rng(seed)
    n_new, src, dst = [list(a) for a in zip(*seqs)]
    x, g, beta = draw(rng, sum(n_new), hk, hv, dk, dv)
    states = rng.normal(0, 0.5, (max(src + dst) + 2, hv, dk, dv)).astype(np.float32)
    if draw is lasting:  # a part of the shortest length leaves a tenth of a state at least
        c = np.concatenate([np.zeros((1, hv)), np.cumsum(g.astype(np.float64), 0)])
        assert (c[part:] - c[:-part]).min() > np.log(0.1)
    print(f"[gpu] delta lasting {hk}/{hv} x {dk}, {dv} {seqs}", flush=True)
    y, s = go(hqlib, x, g, beta, states, n_new, src, dst, hk, hv, dk, dv)
    q, k, v = split(x, hk, hv, dk, dv)
    for h in heads:
        one, kh = slice(h, h + 1), slice(h // (hv // hk), h // (hv // hk) + 1)
        before = [states[i][one] if i >= 0 else np.zeros((1, dk, dv), np.float32) for i in src]
        want, bound, after, e = delta(q[:, kh], k[:, kh], v[:, one], g[:, one], beta[:, one], before, n_new, dk ** -0.5)
        assert (np.abs(y[:, one] - want) <= bound).all(), h
        once = np.sqrt(((want.astype(np.float16).astype(np.float64) - want) ** 2).mean())
        size = 2.0 ** -20 * np.sqrt(max(n_new) / 64)
        assert np.sqrt(((y[:, one] - want) ** 2).mean()) <= 1.1 * once + size * np.sqrt((want * want).mean()), h
        for i_seq, (i, n, a, b) in enumerate(zip(dst, n_new, after, e)):
            if i >= 0:
                assert (np.abs(s[i][one] - a) <= b + U_MIN).all(), h
                if n > 2 * part:  # (what came before the last two parts counts: without it the state is another one)
                    at = slice(sum(n_new[:i_seq + 1]) - 2 * part, sum(n_new[:i_seq + 1]))
                    _, _, last, _ = delta(q[at, kh], k[at, kh], v[at, one], g[at, one], beta[at, one], [np.zeros_like(a)], [2 * part], 1.0)
                    assert np.sqrt(((last[0] - a) ** 2).mean()) > 0.01 * np.sqrt((a * a).mean()), h
                assert np.sqrt(((s[i][one] - a) ** 2).mean()) <= max(2.0 ** -19, 2.0 ** -20 * np.sqrt(n / 64)) * np.sqrt((a * a).mean()) + U_MIN, h


@pytest.mark.parametrize("hk,hv,dk,dv,seqs,heads", [
    (1, 3, 128, 128, [(2000, 0, 1)], (0, 1, 2)),                        # eight parts and more of one sequence
    (1, 3, 64, 128, [(1300, 0, 0), (1100, 1, 2), (30, 3, 3)], (0, 2)),  # of two, a short one beside them
    (3, 3, 128, 48, [(1500, -1, 0)], (0, 1)),                           # from nothing, fewer values than keys
    (1, 2, 256, 96, [(1200, 0, 1)], (0, 1)), (2, 2, 48, 256, [(1700, 1, 0)], (0, 1)),
    (32, 64, 64, 64, [(1280, 0, 0)], (0, 1, 63)),                       # heads enough for one run of 20 chunks
    (32, 64, 64, 64, [(4096, 0, 1)], (0, 2, 61)),                       # and for parts of 22
    (16, 96, 128, 32, [(1500, 0, 1), (1400, 2, 2)], (0, 95))])
def test_states_that_last(hqlib, hk, hv, dk, dv, seqs, heads):
    compare(hqlib, dk + dv + hv, hk, hv, dk, dv, seqs, heads)


def pass_chunks(hv):
    """Chunks of a pass of the workspace, as hq_scan_set has them."""
    h, c = open(os.path.join(CSRC, "hq_scan.h")).read(), open(os.path.join(CSRC, "hq_scan.hip")).read()
    kb = int(re.search(r"HQ_CHUNK_BYTES = (\d+) \* 1024;", h).group(1))
    mb = int(re.search(r"MOST_WORK = \(size_t\)(\d+) << 20;", c).group(1))
    least = int(re.search(r"std::max<size_t>\((\d+), MOST_WORK / per_chunk\)", c).group(1))
    assert "constexpr int HQ_CHUNK = 64;" in h
    return max(least, (mb << 20) // (hv * kb * 1024))


@pytest.mark.parametrize("hk,hv,passes", [(64, 512, 2), (64, 512, 4), (8, 64, 2)])
def test_states_that_last_from_pass_to_pass(hqlib, hk, hv, passes):
    """A sequence over several passes (of the workspace's size as it is), a shorter one before it and one behind it."""
    n = 64 * (passes - 1) * pass_chunks(hv) + 100
    compare(hqlib, hv + passes, hk, hv, 16, 16, [(70, 0, 0), (n, 1, 2), (200, -1, 3)], (0, hv - 1))


@pytest.mark.parametrize("what", ["edges", "one_end", "full", "no_keys"])
def test_edges_in_parts(hqlib, what):
    """Parts where decays of nothing end a state, of everything keep it, with full strengths and with keys of zeros."""
    def change(x, g, beta, states):
        if what == "edges":
            g[::7], g[1::7], g[2::7], g[64:70] = -np.inf, 0, -1e4, -np.inf
            beta[::5], beta[1::5] = 0, 1
            x[3::11, :256] = 0
        elif what == "one_end":  # within a middle part, states last but for one token
            g[:], beta[:] = -1e-3, 0.02
            g[700] = -np.inf
        elif what == "full":  # one key in each part, written with full strength and never decayed
            g[:], beta[:] = 0, 1
            x[:, 128:256] = x[np.arange(len(x)) // 100 * 100, 128:256]
        else:
            g[:], beta[:] = -1e-3, 0.5
            x[:, 128:256] = 0
    check(hqlib, 70, 1, 2, 128, 128, [(1500, 0, 1), (20, 2, 2)], change=change)


def test_describing_a_long_step_among_many(hqlib):
    """One sequence of 2^20 tokens and 60000 of 17: the parts' length is found by halving, so that describing the step takes some twenty looks over the
    sequences and not thousands. Twice as many tokens in the long one are one look more, not twice as many."""
    import time
    print("[gpu] a long step's description", flush=True)
    many, st = 60000, hqlib.States(1, 1, 16, 16, 1, 1, None, None)
    scan = hqlib.Scan(many + 1, (1 << 22) + 17 * many)

    def seconds(n):
        n_new, none = [n] + [17] * many, [-1] * (many + 1)
        n_new, none = np.array(n_new, np.int32), np.array(none, np.int32)
        best = np.inf
        for _ in range(4):
            t = time.process_time()
            scan.set(st, n_new, none, none)
            best = min(best, time.process_time() - t)
        return best
    seconds(1 << 22)
    few, more = seconds(1 << 19), seconds(1 << 22)
    assert more < 4 * few + 0.1 and more < 1.0, (few, more)
    scan.free()
