"""hq_attention where its 16-bit operands come near their ends, against float64 softmax attention (tests/serve_ref.py).

Kernels: single tokens and few rows (k_stream), chunks of rows (k_rows) behind tiles that all of them see and within tiles
that only some do."""
import numpy as np
import pytest

from serve_ref import Pool, attention
from test_gpu_paged_attention import check, run

pytestmark = pytest.mark.gpu


# heads, head_dim, (new, total): single tokens, a few, 128 and 256 rows in several parts and in one
RANGE = [(2, 64, (1, 400)), (4, 128, (7, 130)), (9, 256, (1, 700)), (2, 96, (40, 300)), (4, 128, (130, 700)), (2, 192, (33, 90)), (1, 256, (70, 600))]


@pytest.mark.parametrize("cancel", [False, True])
@pytest.mark.parametrize("nh,hd,lens", RANGE)
@pytest.mark.parametrize("scale", [300, 600, 1024, 30000, 65500])
def test_q8_value_scales_over_their_range(hqlib, scale, nh, hd, lens, cancel):
    """Values of a Q8 cache are code * scale for every finite scale: large ones beside small weights, and (cancel) two large
    ones of equal keys and opposite signs. The bound of serve_ref holds: the operands' roundings with these values' sizes."""
    rng = np.random.default_rng(hd + scale)
    new, n = lens
    far = [3, n // 2, n - 1]  # positions with large scales: one that every row sees, others within or behind the new tokens
    base = rng.normal(0, 1, hd)
    base *= 4 / np.linalg.norm(base)
    q = np.broadcast_to(base, (new, nh, hd)) + rng.normal(0, 0.02, (new, nh, hd))
    k = rng.normal(0, 0.02, (n, 1, hd)) + base / 16  # scores near 1
    k[far] = -0.375 * base                           # near -6: weights of e^-7
    v = rng.normal(0, 1, (n, 1, hd))
    v[far] = rng.uniform(-1, 1, (3, 1, hd))
    v[far, 0, ::7] = 1
    v[far] *= 127 * np.float32(np.float16(scale))
    if cancel:
        k[[5, 6]] = base / 16
        v[[5, 6]] = np.abs(v[far[0]]) * np.array([1, -1])[:, None, None]
    pool = Pool(rng, [n], 16, 1, hd, True)
    pool.put(0, np.arange(n), k.astype(np.float32), v.astype(np.float32))
    assert np.isfinite(pool.get("v", 0, n)).all() and pool.d["v"][pool.table[0, 0], 0, 3] == np.float16(scale)
    q = q.astype(np.float16)
    want, bound = attention(pool, q, [new], [n], 1.0)
    assert np.abs(want).max() < 6e4
    print(f"[gpu] Q8 value scale {scale}: {nh} heads x {hd} {lens} cancel={cancel}", flush=True)
    check(run(hqlib, pool, nh, [lens], q, 1.0), want, bound)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("nh,hd,lens", [(1, 64, (1, 9000)), (8, 128, (2, 3000)), (3, 256, (1, 5000)), (2, 96, (40, 3000)), (4, 128, (70, 2000)), (1, 256, (60, 3000))])
@pytest.mark.parametrize("bits", [13, 17, 21, 25.1])
def test_light_tails(hqlib, bits, nh, hd, lens, q8):
    """One position in 97 has nearly all of the weight, the others 2^-bits of it each, and some dims' values are 0 at the heavy
    ones: those outputs are the tail's alone. Beside serve_ref's bound a weight may be off by half of fp16's subnormal step in
    units of the row's largest, which is 2^6 when it is rounded: 2^-31, in the outputs' sums and in the sum of weights."""
    rng = np.random.default_rng(hd + int(bits))
    new, n = lens
    heavy = np.arange(n) % 97 == 5
    base = np.zeros(hd)
    base[::4] = 1
    q = np.broadcast_to(2 * base, (new, nh, hd)).astype(np.float16)
    top = bits * np.log(2) / (2 * base.sum())  # of a heavy key's dims: its score is bits * ln 2, the others' are near 0
    k = np.where(heavy[:, None, None], top * base, 0) + rng.normal(0, 0.2 / np.sqrt(hd), (n, 1, hd)) * base
    v = rng.uniform(0.5, 1, (n, 1, hd))
    v[heavy, :, :hd // 2] = 0
    pool = Pool(rng, [n], 16, 1, hd, q8)
    pool.put(0, np.arange(n), k.astype(np.float16), v.astype(np.float16))
    want, bound = attention(pool, q, [new], [n], 1.0)
    seen = n - new + 1 + np.arange(new)[:, None, None]
    bound += 2.0 ** -31 * seen / (seen // 97) * (np.abs(v).max() + np.abs(want))
    print(f"[gpu] light tails: 2^-{bits}, {nh} heads x {hd} {lens} q8={q8}", flush=True)
    check(run(hqlib, pool, nh, [lens], q, 1.0), want, bound)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("nh,hd,lens", [(1, 64, (1, 900)), (8, 128, (2, 3000)), (3, 256, (1, 500)), (2, 96, (40, 300)), (4, 128, (70, 2000)), (1, 256, (60, 700))])
@pytest.mark.parametrize("order", ["up", "down", "mixed"])
@pytest.mark.parametrize("scale", [3e5, -1e9, 1e20])
def test_large_scores(hqlib, scale, order, nh, hd, lens, q8):
    """Scores whose fp32 steps are many powers of two of a weight: the row's largest ones share all of it, whatever their size.
    Scores here are exact in fp32 and 10^5 apart at least, so the weights are equal or 0: outputs are off by the weights' and
    their own rounding, and the sums'."""
    rng = np.random.default_rng(hd)
    new, n = lens
    c = rng.integers(-2000, 2001, n)
    c = np.sort(c) if order == "up" else np.sort(c)[::-1] if order == "down" else c
    c[rng.integers(0, n, 4)] = c.max()
    c[rng.integers(0, n, 4)] = c.min()
    k = np.zeros((n, 1, hd), np.float16)
    k[:, 0, 3] = c
    q = np.zeros((new, nh, hd), np.float16)
    q[:, :, 3] = 1
    pool = Pool(rng, [n], 16, 1, hd, q8)
    pool.put(0, np.arange(n), k, rng.normal(0, 1, (n, 1, hd)).astype(np.float16))
    want, _ = attention(pool, q, [new], [n], scale)
    v = np.abs(pool.get("v", 0, n)).max()
    print(f"[gpu] large scores: {scale} {order}, {nh} heads x {hd} {lens} q8={q8}", flush=True)
    check(run(hqlib, pool, nh, [lens], q, scale), want, np.full(want.shape, 3 * 2.0 ** -11 * v))
