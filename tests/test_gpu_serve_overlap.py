"""Work of two streams at a time: all of it is queued before the first wait, and each stream's calls have shapes of their own, so that memory which
the library kept for both would be written by one while the other reads it. Results are the bits of the same calls alone."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


class Recurrent:
    """A step of a recurrent layer (append, recurrence) on a stream and a description of its own."""

    def __init__(self, hqlib, seed, hk, hv, dk, dv, n_new, gated):
        rng = np.random.default_rng(seed)
        self.hq, self.stream, n, T, taps = hqlib, hqlib.Stream(), len(n_new), sum(n_new), 4
        self.C, up = 2 * hk * dk + hv * dv, hqlib.DevBuf.from_array
        self.x, self.ab = up(rng.normal(0, 1, (T, self.C)).astype(np.float16)), up(rng.normal(0, 1, (2, T, hv)).astype(np.float16))
        self.w, self.al, self.dt = up(rng.normal(0, 0.5, (self.C, taps)).astype(np.float32)), up(rng.uniform(-6, -3, hv).astype(np.float32)), up(rng.normal(0, 1, hv).astype(np.float32))
        self.s, self.conv = up(rng.normal(0, 0.3, (2 * n, hv, dk, dv)).astype(np.float32)), up(rng.normal(0, 1, (2 * n, taps - 1, self.C)).astype(np.float32))
        self.out = [hqlib.DevBuf(b) for b in (T * self.C * 2, T * hv * 4, T * hv * 4, T * hv * dv * 2)]
        self.st, self.scan = hqlib.States(hk, hv, dk, dv, taps, 2 * n, self.s, self.conv), hqlib.Scan(n, T)
        self.scan.set(self.st, n_new, np.arange(n), np.arange(n, 2 * n), stream=self.stream.ptr)
        self.b = self.ab.ptr + T * hv * 2
        self.at = [2 * hk * dk, 4 * hk * dk]
        self.kw = dict(norm=up(np.ones(dv, np.float32)), gate=up(rng.normal(0, 1, (T, hv * dv)).astype(np.float32)), gate_f32=True) if gated else {}
        self.scale = dk ** -0.5

    def run(self):
        qkv, g, beta, o = self.out
        self.hq.delta_append(self.scan, self.st, self.x, self.w, self.ab, self.b, self.al, self.dt, qkv, g, beta, f32=False, stream=self.stream.ptr)
        self.hq.delta(self.scan, self.st, qkv, qkv.ptr + self.at[0], qkv.ptr + self.at[1], g, beta, o, self.scale, qk_stride=self.C, v_stride=self.C,
                      stream=self.stream.ptr, **self.kw)

    def results(self):
        return [b.download((b.nbytes,), np.uint8) for b in (*self.out, self.s, self.conv)]

    def free(self):
        self.scan.free()
        self.stream.destroy()


class Choice:
    """A beam step and log probabilities on a stream of their own."""

    def __init__(self, hqlib, seed, G, B, V, k):
        rng = np.random.default_rng(seed)
        self.hq, self.stream, self.shape, self.k = hqlib, hqlib.Stream(), (G, B, V), k
        self.x, self.score = hqlib.DevBuf.from_array(rng.normal(0, 3, (G * B, V)).astype(np.float32)), hqlib.DevBuf.from_array(rng.normal(-9, 3, G * B).astype(np.float32))
        self.out = [hqlib.DevBuf(G * k * 4) for _ in range(3)] + [hqlib.DevBuf(G * B * 4), hqlib.DevBuf(G * B * k * 4), hqlib.DevBuf(G * B * k * 4)]

    def run(self):
        G, B, V = self.shape
        self.hq.beam(self.x, G, B, V, self.score, self.k, *self.out[:3], f32=True, stream=self.stream.ptr)
        self.hq.logprobs(self.x, G * B, V, f32=True, top_k=self.k, entropy=self.out[3], top_ids=self.out[4], top_logp=self.out[5], stream=self.stream.ptr)

    def results(self):
        return [b.download((b.nbytes,), np.uint8) for b in self.out]

    def free(self):
        self.stream.destroy()


def side_by_side(hqlib, work):
    want = []
    for w in work:
        w.run()
        w.stream.sync()
        want.append(w.results())
    for _ in range(4):
        for w in work:
            for b in w.out:
                b.upload(np.full(b.nbytes, 0xa5, np.uint8))
        hqlib.synchronize()
        for _ in range(6):
            for w in work:
                w.run()
        for w in work:
            w.stream.sync()
        for w, r in zip(work, want):
            assert all(np.array_equal(a, b) for a, b in zip(w.results(), r))
    for w in work:
        w.free()


def test_recurrent_steps(hqlib):
    print("[gpu] recurrent steps on three streams", flush=True)
    side_by_side(hqlib, [Recurrent(hqlib, 1, 2, 4, 128, 128, [3000, 5, 1], True), Recurrent(hqlib, 2, 1, 2, 64, 96, [1, 4000, 70], True),
                         Recurrent(hqlib, 3, 16, 32, 64, 64, [1] * 40 + [7] * 9, False)])


def test_choices(hqlib):
    print("[gpu] choices on three streams", flush=True)
    side_by_side(hqlib, [Choice(hqlib, 4, 1, 4, 151936, 8), Choice(hqlib, 5, 40, 3, 30011, 6), Choice(hqlib, 6, 3, 7, 90000, 20)])


def test_both(hqlib):
    print("[gpu] a recurrent step and choices", flush=True)
    side_by_side(hqlib, [Recurrent(hqlib, 7, 1, 2, 64, 64, [2500, 1, 30], True), Choice(hqlib, 8, 2, 8, 100003, 16), Recurrent(hqlib, 9, 4, 4, 32, 32, [900, 800], False)])
