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
