"""hip_batch_step (include/hq_backend.h): sequences of different lengths through a whole model over the paged cache, step by
step (prompts, chunks, single tokens, sequences that join and rest), against a float64 forward of each sequence by itself.

Tolerances: the logits' bar of every forward test is 1e-2 (GEMM operands rounded to fp16, logits of size ~1), and a log
probability is a logit less a mean of logits of the same row, so 2e-2. A Q8 cache is off by up to 1/254 of a head's largest
value, 0.7 % of its size in the root mean square; through two layers' attention that is up to 2e-2 of logits of size ~1 at the
worst of 512, and twice that of log probabilities: 6e-2 in all. A page, position, gate or norm read from a wrong place is
another vector of order 1.
"""
import numpy as np
import pytest

import synth
from test_gpu_backend_options import MIXED, Q4, Q8, forward64, make

pytestmark = pytest.mark.gpu
VOCAB = 512


def log_softmax(x):
    m = x.max(-1, keepdims=True)
    return x - m - np.log(np.exp(x - m).sum(-1, keepdims=True))


CASES = [  # types, gate, q/k norm, offset, heads, kv heads, head size, rotated dims, page size, Q8 cache
    (Q8, True, True, 1.0, 4, 2, 64, 32, 16, False), (MIXED, False, True, 0.0, 4, 1, 128, 64, 32, False), (Q4, False, False, 0.0, 8, 8, 64, 64, 64, True),
    (Q8, True, False, 0.0, 4, 4, 96, 96, 16, True), (MIXED, True, True, 1.0, 2, 1, 256, 64, 16, False)]


@pytest.mark.parametrize("types,gate,qk_norm,offset,nh,nkv,hd,rot,page,q8", CASES)
def test_steps(hqlib, oracle, types, gate, qk_norm, offset, nh, nkv, hd, rot, page, q8):
    print(f"[gpu] batch steps gate={gate} qk_norm={qk_norm} {nh}/{nkv} x {hd} page {page} q8={q8}", flush=True)
    model = make(nh + hd + page, types, gate, qk_norm, offset, nh, nkv, hd, rot)
    be = hqlib.HipBackend(hqlib.RefModelView(model), 64)
    first = be.forward(np.arange(40), np.arange(16))
    max_pages = 256 // page
    n_pages = 4 * max_pages + 3
    s = hqlib.HipBatch(be, n_pages, page, 4, 300, max_pages, hqlib.KV_Q8 if q8 else hqlib.KV_F16)
    rng = synth.Rng(page + hd)
    seqs = [rng.integers(0, VOCAB - 1, 256).astype(np.uint32) for _ in range(4)]
    pages = rng.choice_without_replacement(n_pages, 4 * max_pages).astype(np.uint32).reshape(4, max_pages)
    every = np.tile(np.arange(VOCAB, dtype=np.uint32), (4, 1))
    pos = np.zeros(4, np.int64)
    worst = 0.0
    # prompts; chunks and a single token and a new sequence; single tokens; one token alone; a long chunk next to single tokens
    for n_new in ([70, 33, 1, 0], [17, 1, 0, 129], [1, 1, 1, 1], [0, 1, 0, 0], [1, 150, 2, 1]):
        pos += n_new
        tokens = np.concatenate([t[p - n:p] for t, p, n in zip(seqs, pos, n_new)])
        logp, entropy, top_ids, top_logp = s.step(tokens, n_new, pos, pages, every, 5)
        for i in range(4):
            if not n_new[i]:
                assert np.isnan(logp[i]).all() and np.isnan(entropy[i])
                continue
            logits = forward64(oracle, hqlib, model, seqs[i][:pos[i]], every[0])
            want = log_softmax(logits)
            assert np.abs(logits).max() > 0.1
            worst = max(worst, np.abs(logp[i] - want).max())
            # what is asked of the same row agrees with itself
            got = logp[i].astype(np.float64)
            assert np.array_equal(top_ids[i], np.lexsort((np.arange(VOCAB), -logp[i]))[:5])
            assert np.abs(top_logp[i] - got[top_ids[i]]).max() <= 1e-6
            assert abs(entropy[i] + (np.exp(got) * got).sum()) <= 1e-4
    print(f"[gpu]   log probabilities off by {worst:.2e}", flush=True)
    assert worst <= (6e-2 if q8 else 2e-2)
    s.free()
    # the backend's own state is its own
    be.reset()
    assert np.array_equal(be.forward(np.arange(40), np.arange(16)), first)
    be.destroy()


def test_refusals(hqlib):
    model = make(5, Q8, False, False, 0.0, 4, 2, 64, 64)
    be = hqlib.HipBackend(hqlib.RefModelView(model), 64)
    for kw, text in ((dict(page_size=24), "page_size 24"), (dict(n_pages=0), "0 pages"), (dict(max_tokens=0), "0 tokens"), (dict(max_seqs=0), "0 sequences"),
                     (dict(max_pages=0), "0 a sequence"), (dict(kv_type=2), "cache type 2")):
        with pytest.raises(hqlib.HQError, match=text):
            hqlib.HipBatch(be, **{**dict(n_pages=8, page_size=16, max_seqs=2, max_tokens=32, max_pages=4), **kw})
    s = hqlib.HipBatch(be, 8, 16, 2, 32, 4)
    pages = np.arange(8).reshape(2, 4)
    ok = dict(tokens=np.arange(5), n_new=[3, 2], n_pos=[3, 2], pages=pages)
    for kw, text in ((dict(tokens=[1, 2, 3, 4, VOCAB]), "token 512"), (dict(n_pos=[2, 2]), "3 new tokens of 2"), (dict(pages=pages + 4), "page 0 of sequence 1 is 8"),
                     (dict(n_pos=[65, 2]), "needs 5 pages"), (dict(tokens=np.arange(40), n_new=[38, 2], n_pos=[38, 2]), "40 new tokens"),
                     (dict(ids=[[1], [VOCAB]]), "id 512"), (dict(top_k=65), "top_k 65"),
                     (dict(tokens=np.arange(3), n_new=[1, 1, 1], n_pos=[1, 1, 1], pages=np.arange(3).reshape(3, 1)), "3 sequences")):
        with pytest.raises(hqlib.HQError, match=text):
            s.step(**{**ok, **kw})
    # a refused step leaves the batch usable; a step of nothing is one
    a = s.step(**ok, top_k=3)
    s.step([], [0, 0], [0, 0], pages)
    b = s.step(**ok, top_k=3)
    assert all(np.array_equal(x, y) for x, y in zip(a, b))
    s.free()
    be.destroy()
    odd = make(6, Q8, False, False, 0.0, 4, 2, 72, 64)
    be = hqlib.HipBackend(hqlib.RefModelView(odd), 64)
    with pytest.raises(hqlib.HQError, match="head_dim 72"):
        hqlib.HipBatch(be, 8, 16, 2, 32, 4)
    be.destroy()
