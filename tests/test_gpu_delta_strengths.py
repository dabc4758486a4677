"""hq_delta where write strengths are small as a whole. A state that begins with zeros is then small too, and as exact relative to itself as
one of full strengths: a state's operands are two fp16 terms each, good to 2^-22 of their column's largest, and the 64 x 64 matrix of a chunk's
writes likewise, of its largest entry. Errors of many operands are independent: in the root mean square the state is within 2^-19 of its own
size (test_gpu_delta.check), and outputs within 1.1 times what their one rounding to fp16 makes (1.1^2 - 1 leaves the rest 0.46 of it, some 2^-13)."""
import numpy as np
import pytest

from delta_ref import delta
from test_gpu_delta import U_MIN, go, inputs, split

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hk,hv,dk,dv,seqs", [
    (1, 2, 128, 128, [(64, -1, 0), (300, -1, 1)]), (1, 1, 64, 64, [(1300, -1, 0)]), (1, 1, 256, 48, [(130, -1, 0)]), (1, 2, 32, 128, [(12, -1, 0), (8, -1, 1), (90, -1, 2)])])
@pytest.mark.parametrize("strength", [1.0, 2.0 ** -10, 2.0 ** -15, 2.0 ** -20, 2.0 ** -30, 2.0 ** -60, 2.0 ** -80])
def test_small_strengths(hqlib, hk, hv, dk, dv, seqs, strength):
    rng = np.random.default_rng(hv + dk)
    n_new, src, dst = [list(a) for a in zip(*seqs)]
    x, g, beta = inputs(rng, sum(n_new), hk, hv, dk, dv)
    beta *= np.float32(strength)
    states = np.zeros((max(dst) + 2, hv, dk, dv), np.float32)
    print(f"[gpu] delta strengths of {strength} {hk}/{hv} x {dk}, {dv} {seqs}", flush=True)
    scale = float(np.float32(min(dk ** -0.5 / strength, 1e20)))
    y, s = go(hqlib, x, g, beta, states, n_new, src, dst, hk, hv, dk, dv, scale=scale)
    want, bound, after, e = delta(*split(x, hk, hv, dk, dv), g, beta, [np.zeros((hv, dk, dv), np.float32)] * len(n_new), n_new, scale)
    for i, a in zip(dst, after):
        assert np.sqrt(((s[i] - a) ** 2).mean()) <= 2.0 ** -19 * np.sqrt((a * a).mean()) + U_MIN
    once = np.sqrt(((want.astype(np.float16).astype(np.float64) - want) ** 2).mean())
    assert np.sqrt(((y - want) ** 2).mean()) <= 1.1 * once


def test_one_strong_token_among_weak_ones(hqlib):
    """Strengths that differ by 2^20 within a chunk, the strong token at its start, middle and end, and nothing written at all."""
    hk, hv, dk, dv, n = 1, 1, 64, 64, 256
    rng = np.random.default_rng(3)
    x, g, beta = inputs(rng, n, hk, hv, dk, dv)
    beta *= np.float32(2.0 ** -20)
    beta[[0, 100, 191]] = 1
    beta[192:] = 0
    states = rng.normal(0, 0.5, (2, hv, dk, dv)).astype(np.float32)
    print("[gpu] delta one strong token", flush=True)
    y, s = go(hqlib, x, g, beta, states, [n], [0], [1], hk, hv, dk, dv)
    want, bound, after, e = delta(*split(x, hk, hv, dk, dv), g, beta, [states[0]], [n], dk ** -0.5)
    assert (np.abs(y - want) <= bound).all() and (np.abs(s[1] - after[0]) <= e[0] + U_MIN).all()
    assert np.sqrt(((s[1] - after[0]) ** 2).mean()) <= 2.0 ** -19 * np.sqrt((after[0] * after[0]).mean()) + U_MIN
