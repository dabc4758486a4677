"""Beam search over a model: hip_batch_beam, hip_batch_copy and hq_pages together (include/hq_backend.h, include/hq_serve.h), each step
against float64 forwards of every beam's whole history; and the same over a layer with a recurrent state, whose slots the beams
branch between.

Tolerances: a step's log probabilities are within those of a whole forward test, 2e-2 with an fp16 cache and 6e-2 with a Q8 one
(tests/test_gpu_batch.py); a choice may differ from float64's where the values are nearer than twice that."""
import numpy as np
import pytest

import delta_ref
import synth
from test_gpu_backend_options import MIXED, Q8, forward64, make

pytestmark = pytest.mark.gpu
VOCAB, EOS = 512, 7


def log_softmax(x):
    m = x.max(-1, keepdims=True)
    return x - m - np.log(np.exp(x - m).sum(-1, keepdims=True))


def check_choice(want, score, done, got, tol, eos):
    """want [beams, vocab]: log probabilities of the beams that are read. got: (score, token, beam) [k] of one group."""
    value = score[:, None].astype(np.float64) + want
    for b in range(len(score)):
        if done[b]:
            value[b] = -np.inf
            value[b, eos] = score[b]
        elif score[b] == -np.inf:
            value[b] = -np.inf
    s, t, b = got
    k = int(np.isfinite(value).sum(initial=0))
    n = min(len(s), k)
    assert (b[n:] == -1).all() and (s[n:] == -np.inf).all()
    assert len(set(zip(t[:n].tolist(), b[:n].tolist()))) == n and (np.diff(s[:n]) <= 0).all()
    chosen = value[b[:n], t[:n]]
    assert np.isfinite(chosen).all() and np.abs(s[:n] - chosen).max() <= tol
    value[b[:n], t[:n]] = -np.inf
    assert value.max() <= s[n - 1] + 2 * tol
    return np.abs(s[:n] - chosen).max()


@pytest.mark.parametrize("types,gate,nh,nkv,hd,rot,page,q8", [(Q8, False, 4, 2, 64, 64, 16, False), (MIXED, True, 4, 1, 128, 64, 16, True)])
def test_search(hqlib, oracle, types, gate, nh, nkv, hd, rot, page, q8):
    print(f"[gpu] beam search {nh}/{nkv} x {hd} q8={q8}", flush=True)
    model = make(nh + hd, types, gate, True, 0.0, nh, nkv, hd, rot)
    be = hqlib.HipBackend(hqlib.RefModelView(model), 64)
    G, B, steps, max_pages, n_pages = 3, 4, 20, 6, 40
    tol = 6e-2 if q8 else 2e-2
    s = hqlib.HipBatch(be, n_pages, page, G * B, 128, max_pages, hqlib.KV_Q8 if q8 else hqlib.KV_F16)
    pages = hqlib.Pages(n_pages, page, 2 * G * B)  # a step's beams, and those they come from
    rng = synth.Rng(hd)
    prompts = [rng.integers(0, VOCAB - 1, n).astype(np.uint32) for n in (1, 15, 45)]
    now, then = np.arange(G * B), np.arange(G * B, 2 * G * B)
    # the prompts, to the first beam of each group; the others have not begun
    text = [[list(p)] + [[] for _ in range(B - 1)] for p in prompts]
    score = np.full((G, B), -np.inf, np.float32)
    score[:, 0] = 0
    done = np.zeros((G, B), np.uint8)
    n_new = np.zeros((G, B), np.int32)
    n_new[:, 0] = [len(p) for p in prompts]
    n_pos = n_new.copy()
    for i in range(G):
        pages.resize(now[i * B], 0, n_pos[i, 0])
    tokens = np.concatenate(prompts)
    worst, copied, shared = 0.0, 0, 0
    for step in range(steps):
        src, dst, n = pages.copies()
        copied += len(src)
        s.copy(src, dst, n)
        table = pages.table(now, max_pages)
        got = s.beam(tokens, n_new.ravel(), n_pos.ravel(), table, score, B, done, EOS)
        for i in range(G):
            want = np.full((B, VOCAB), -np.inf)
            for b in range(B):
                if not done[i, b] and score[i, b] > -np.inf:
                    want[b] = log_softmax(forward64(oracle, hqlib, model, np.array(text[i][b]), np.arange(VOCAB)))
            worst = max(worst, check_choice(want, score[i], done[i], [a[i] for a in got], tol, EOS))
        # the beams go on from where they come from
        new_text = [[text[i][b] + ([] if done[i, b] else [int(t)]) for t, b in zip(got[1][i], got[2][i])] for i in range(G)]
        was, come = n_pos, got[2]
        ended = np.take_along_axis(done, come, 1)
        n_pos = np.take_along_axis(was, come, 1)
        for i in range(G):
            for b in range(B):
                pages.fork(now[i * B + come[i, b]], then[i * B + b], int(n_pos[i, b]))
        for q in now:
            pages.resize(q, 0, 0)
        now, then = then, now
        score, text = got[0], new_text
        done = np.where(ended | (got[1] % 64 == EOS) | (n_pos + 1 > max_pages * page), 1, 0).astype(np.uint8)
        n_new = np.where(ended, 0, 1).astype(np.int32)  # (the token that ends a beam is still taken in)
        n_pos = n_pos + n_new
        for i in range(G):
            for b in range(B):
                pages.resize(now[i * B + b], int(n_pos[i, b] - n_new[i, b]), int(n_pos[i, b]))
        tokens = np.array([text[i][b][-1] for i in range(G) for b in range(B) if n_new[i, b]], np.uint32)
        if step % 7 == 3:
            src, dst, n = pages.copies()
            copied += len(src)
            s.copy(src, dst, n)
            pages.compact()
        t = pages.table(now, max_pages)
        held = [t[j, :-(-int(p) // page)] for j, p in enumerate(n_pos.ravel())]
        shared = max(shared, sum(map(len, held)) - len(set(np.concatenate(held).tolist())))
    print(f"[gpu]   scores off by {worst:.2e}, {copied} pages copied, {shared} shared, {int(done.sum())} beams ended", flush=True)
    assert copied > 10 and shared > 3
    pages.copies()
    for q in now:
        pages.resize(q, 0, 0)
    assert pages.count()[1] == n_pages
    s.free()
    be.destroy()


def test_steps_of_nothing_and_refusals(hqlib):
    model = make(5, Q8, False, False, 0.0, 4, 2, 64, 64)
    be = hqlib.HipBackend(hqlib.RefModelView(model), 64)
    s = hqlib.HipBatch(be, 8, 16, 4, 3, 4)  # (more sequences than tokens of a step)
    pages = np.arange(8, dtype=np.uint32).reshape(4, 2)
    no = -np.inf
    ok = dict(tokens=[1, 2, 3], n_new=[2, 0, 1, 0], n_pos=[2, 0, 1, 0], pages=pages, score=[[0, no], [-1, -2]], k=3, done=[[0, 0], [0, 1]], done_token=9)
    a = s.beam(**ok)
    assert (a[2][0] == 0).all() and 1 in a[2][1] and a[1][1][list(a[2][1]).index(1)] == 9
    for kw, text in ((dict(tokens=[1, 2, VOCAB]), "token 512"), (dict(n_pos=[1, 0, 1, 0]), "2 new tokens of 1"), (dict(pages=pages + 7), "page 0 of sequence 2 is 11|is 8"),
                     (dict(k=0), "k 0"), (dict(k=65), "k 65"), (dict(score=[[0, -1], [-1, -2]]), "beam 1 of group 0 has no new tokens"),
                     (dict(done=None), "beam 1 of group 1 has no new tokens"), (dict(n_new=[2, 0, 2, 0], n_pos=[2, 0, 2, 0], tokens=[1, 2, 3, 4]), "4 new tokens"),
                     (dict(score=np.zeros((5, 1)), done=None, n_new=[1, 1, 1, 0, 0], n_pos=[1] * 5, pages=np.zeros((5, 2))), "5 groups of 1")):
        with pytest.raises(hqlib.HQError, match=text):
            s.beam(**{**ok, **kw})
    for args, text in ((([8], [0]), "page 8"), (([0], [8]), "page 8"), (([0, 1], [2, 2]), "two copies"), (([0, 1], [1, 2]), "page 1"), (([0], [1], [17]), "17 positions")):
        with pytest.raises(hqlib.HQError, match=text):
            s.copy(*args)
    s.copy([], [])
    b = s.beam(**ok)
    assert all(np.array_equal(x, y) for x, y in zip(a, b))
    # nobody goes on: done beams stay, and nothing is run
    got = s.beam([], [0] * 4, [2, 0, 1, 0], pages, [[0, no], [-1, -2]], 3, [[1, 1], [1, 1]], 9)
    assert got[0].tolist() == [[0, no, no], [-1, -2, no]] and got[1][:, 0].tolist() == [9, 9] and got[2].tolist() == [[0, -1, -1], [0, 1, -1]]
    got = s.beam([], [], [], np.zeros((0, 2)), np.zeros((0, 4)), 3)
    assert all(a.shape == (0, 3) for a in got)
    # a copied page is the page: the same step over it
    a = s.step([4], [1], [3], pages[:1], top_k=4)  # (behind the two tokens of the first beam)
    s.copy([0], [5], [2])
    b = s.step([4], [1], [3], [[5, 1]], top_k=4)
    assert all(np.array_equal(x, y) for x, y in zip(a, b))
    s.free()
    be.destroy()


def test_recurrent_search(hqlib):
    """A layer of gated delta heads between an embedding and the logits: hq_delta_append, hq_delta, hq_gemm and hq_beam in a row,
    beams that go on from each other's slots. The layer's own outputs are held to their bounds by the tests of its operators; the
    logits are products of a matrix of Q8_0 blocks with its fp16 outputs, 2^-11 a term of sums of size ~1 on top, and 2e-2 is asked
    as of a whole model."""
    hk, hv, dk, dv, taps, G, B, steps = 2, 4, 64, 64, 4, 2, 3, 70
    C, rng = 2 * hk * dk + hv * dv, np.random.default_rng(21)
    head = synth.quantize_q8_0(rng.normal(0, 0.06, (VOCAB, hv * dv)).astype(np.float32))
    W = hqlib.Mat(head, synth.Q8_0, VOCAB, hv * dv)
    w64 = head.reshape(-1, 34)
    w64 = (w64[:, :2].copy().view(np.float16).astype(np.float64) * w64[:, 2:].view(np.int8)).reshape(VOCAB, hv * dv)
    emb = rng.normal(0, 1, (VOCAB, C)).astype(np.float32)
    ea, eb, ez = (rng.normal(0, 1, (VOCAB, n)).astype(np.float32) for n in (hv, hv, hv * dv))
    conv, a_log, dt, norm = rng.normal(0, 0.5, (C, taps)).astype(np.float32), rng.uniform(-3, 0, hv).astype(np.float32), rng.normal(0, 1, hv).astype(np.float32), np.ones(dv, np.float32)
    up = hqlib.DevBuf.from_array
    dS, dC = up(np.full((2 * G * B, hv, dk, dv), np.nan, np.float32)), up(np.full((2 * G * B, taps - 1, C), np.nan, np.float32))
    st = hqlib.States(hk, hv, dk, dv, taps, 2 * G * B, dS, dC)
    scan = hqlib.Scan(G * B, 256)
    const = [up(a) for a in (conv, a_log, dt, norm)]
    out = [hqlib.DevBuf(G * B * 4) for _ in range(3)]

    def layer64(text):
        T = np.array(text)
        qkv, _, g, _, beta, _, _ = delta_ref.append(emb[T], [np.zeros((taps - 1, C))], conv, ea[T], eb[T], a_log, dt, [len(T)], hk, hv, dk, dv, 1e-6)
        c = hk * dk
        o, _, _, _ = delta_ref.delta(qkv[:, :c].reshape(-1, hk, dk), qkv[:, c:2 * c].reshape(-1, hk, dk), qkv[:, 2 * c:].reshape(-1, hv, dv), g, beta,
                                     [np.zeros((hv, dk, dv))], [len(T)], dk ** -0.5, norm, ez[T].reshape(-1, hv, dv), 1e-6)
        return log_softmax(w64 @ o[-1].reshape(-1))

    prompts = [rng.integers(0, VOCAB, n).tolist() for n in (1, 130)]
    text = [[p] + [[] for _ in range(B - 1)] for p in prompts]
    score = np.full((G, B), -np.inf, np.float32)
    score[:, 0] = 0
    n_new = np.array([[len(p)] + [0] * (B - 1) for p in prompts]).ravel()
    slot_from, base, worst = np.full(G * B, -1, np.int32), 0, 0.0
    print("[gpu] recurrent beam search", flush=True)
    for step in range(steps):
        tok = np.concatenate([np.array(text[i][b], np.int64)[len(text[i][b]) - n_new[i * B + b]:] for i in range(G) for b in range(B)])
        T, last = len(tok), np.maximum(np.cumsum(n_new) - 1, 0)
        x, a, b_, z = (up(e[tok]) for e in (emb, ea, eb, ez))
        qkv, g, beta, o = hqlib.DevBuf(T * C * 2), hqlib.DevBuf(T * hv * 4), hqlib.DevBuf(T * hv * 4), hqlib.DevBuf(T * hv * dv * 2)
        scan.set(st, n_new, slot_from, np.arange(G * B) + base)
        hqlib.delta_append(scan, st, x, const[0], a, b_, const[1], const[2], qkv, g, beta, f32=True)
        hqlib.delta(scan, st, qkv, qkv.ptr + 2 * hk * dk, qkv.ptr + 4 * hk * dk, g, beta, o, dk ** -0.5, qk_stride=C, v_stride=C, norm=const[3], gate=z, gate_f32=True)
        hqlib.synchronize()
        rows = up(o.download((T, hv * dv), np.float16)[last])  # (each sequence's last token; a beam that has not begun: any)
        logits, d_score = hqlib.DevBuf(G * B * VOCAB * 4), up(score)
        hqlib.gemm(W, rows, G * B, logits)
        hqlib.beam(logits, G, B, VOCAB, d_score, B, *out, f32=True)
        hqlib.synchronize()
        got = [d.download((G, B), t) for d, t in zip(out, (np.float32, np.uint32, np.int32))]
        if step % 6 == 0 or step > steps - 3:
            for i in range(G):
                want = np.stack([layer64(text[i][b]) if score[i, b] > -np.inf else np.zeros(VOCAB) for b in range(B)])
                worst = max(worst, check_choice(want, score[i], np.zeros(B), [a[i] for a in got], 2e-2, 0))
        text = [[text[i][b] + [int(t)] for t, b in zip(got[1][i], got[2][i])] for i in range(G)]
        slot_from = (got[2] + np.arange(G)[:, None] * B + base).ravel().astype(np.int32)
        base, n_new, score = G * B - base, np.ones(G * B, np.int64), got[0]
    print(f"[gpu]   scores off by {worst:.2e}", flush=True)
    scan.free()
