"""hq_attention: padding tokens (before position 0) give zeros whatever their rows hold, queries and gates of NaN among it, and
leave the tokens behind them alone."""
import numpy as np
import pytest

from serve_ref import Pool, attention, fill
from test_gpu_paged_attention import check, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gate_f32", [False, True])
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("nh,nkv,hd,lens", [(4, 2, 64, [(3, 1), (2, 0), (1, 40)]), (4, 1, 128, [(9, 4), (7, 3000)]), (6, 2, 96, [(40, 7), (70, 60)]),
                                            (16, 4, 256, [(40, 30), (50, 0)]), (8, 1, 64, [(80, 50), (3, 2)])])
def test_padding_rows_of_nan(hqlib, nh, nkv, hd, lens, q8, gate_f32):
    rng = np.random.default_rng(nh + hd)
    n_new, n_pos = [a for a, _ in lens], [t for _, t in lens]
    pool = Pool(rng, n_pos, 16, nkv, hd, q8)
    fill(pool, rng, n_pos)
    T = sum(n_new)
    q, gate = rng.normal(0, 2, (2, T, nh, hd)).astype(np.float16)
    want, bound = attention(pool, q, n_new, n_pos, hd ** -0.5, gate)
    pad = np.concatenate([np.arange(t - a, t) < 0 for a, t in lens])
    assert pad.any() and (want[pad] == 0).all()
    q[pad], gate[pad] = np.nan, np.nan
    print(f"[gpu] padding: {nh}/{nkv} x {hd} {lens} q8={q8} gate_f32={gate_f32}", flush=True)
    got = run(hqlib, pool, nh, lens, q, hd ** -0.5, gate=gate, gate_f32=gate_f32)
    assert (got[pad] == 0).all()
    check(got[~pad], want[~pad], bound[~pad])
