"""hq_beam's order where a beam's values are equal though its logits are not: values are formed in 64 bits, and a difference of logits can be lost
in them next to a large score, or next to the row's largest logit. The larger logit comes first, as the exact values would have it."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def go(hqlib, x, score, k):
    G, B, V = x.shape
    d = [hqlib.DevBuf.from_array(a) for a in (np.ascontiguousarray(x, np.float32), np.ascontiguousarray(score, np.float32))]
    out = [hqlib.DevBuf(G * k * 4) for _ in range(3)]
    hqlib.beam(d[0], G, B, V, d[1], k, *out, f32=True)
    hqlib.synchronize()
    return [o.download((G, k), t) for o, t in zip(out, (np.float32, np.uint32, np.int32))]


@pytest.mark.parametrize("V,k", [(7, 12), (5000, 16)])
@pytest.mark.parametrize("low", [np.finfo(np.float32).min, -1e30, -1e9])
def test_scores_far_below(hqlib, V, k, low):
    """A beam that counts, and two whose scores are far below: they fill the places that it leaves (V 7), beam by beam, each by its logits."""
    print(f"[gpu] beam scores of {low}, {V}", flush=True)
    rng = np.random.default_rng(V)
    x = rng.permutation(V)[None, None] / np.float32(64) + np.zeros((1, 3, 1), np.float32)
    x[0, 1] = x[0, 1, ::-1]
    score, token, beam = go(hqlib, x, [[low, -1, low]], k)
    first = min(V, k)
    assert (beam[0, :first] == 1).all() and np.array_equal(token[0, :first], np.argsort(-x[0, 1], kind="stable")[:first])
    if V < k and low < -1e20:  # (equal values: beam 0 before beam 2; both rows are alike)
        assert (beam[0, first:] == 0).all() and np.array_equal(token[0, first:], np.argsort(-x[0, 0], kind="stable")[:k - first])
        assert (score[0, first:] == np.float32(low)).all()


def test_logits_next_to_zero(hqlib):
    """Logits of 1e-30 and below beside one of 40: their values differ by nothing, their order is theirs."""
    print("[gpu] beam logits next to zero", flush=True)
    V, k = 300, 20
    rng = np.random.default_rng(1)
    x = np.full((1, 1, V), -5, np.float32)
    x[0, 0, 250] = 40
    at = rng.permutation(200)[:30]
    x[0, 0, at] = np.float32(1e-30) * (1 + rng.permutation(30).astype(np.float32) // 2)  # pairs of equal ones
    score, token, beam = go(hqlib, x, [[-0.5]], k)
    assert np.array_equal(token[0], np.lexsort((np.arange(V), -x[0, 0].astype(np.float64)))[:k]) and (beam == 0).all()
    assert len(set(score[0, 1:])) == 1
