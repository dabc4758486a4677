"""The calls of a step with recurrent layers, page copies and beam selection in a captured graph (include/hq_serve.h: they allocate
nothing), replayed between eager work, and two of them side by side on two streams. Every replay gives the eager call's bits."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip(hqlib):
    L = hqlib.load()  # (its dependencies' functions are found through it)
    for f in ("hipStreamBeginCapture", "hipStreamEndCapture", "hipGraphInstantiate", "hipGraphLaunch", "hipGraphDestroy", "hipGraphExecDestroy"):
        getattr(L, f).restype = C.c_int
    return L


class Step:
    """Sequences by chunks in parts, by chunks and token by token through one layer; copies of pages; a beam step. Inputs and the
    states that are read stay as they are, so that the step can be run again."""

    def __init__(self, hqlib, seed, n_new, gated):
        rng = np.random.default_rng(seed)
        self.hq, self.stream = hqlib, hqlib.Stream()
        hk, hv, dk, dv, taps, n, T = 2, 4, 64, 64, 4, len(n_new), sum(n_new)
        self.C, up = 2 * hk * dk + hv * dv, hqlib.DevBuf.from_array
        self.x, self.a, self.b = up(rng.normal(0, 1, (T, self.C)).astype(np.float32)), up(rng.normal(0, 1, (T, hv)).astype(np.float32)), up(rng.normal(0, 1, (T, hv)).astype(np.float32))
        self.z, self.norm = up(rng.normal(0, 1, (T, hv * dv)).astype(np.float16)), up(np.ones(dv, np.float32))
        self.w, self.al, self.dt = up(rng.normal(0, 0.5, (self.C, taps)).astype(np.float32)), up(rng.uniform(-3, 0, hv).astype(np.float32)), up(rng.normal(0, 1, hv).astype(np.float32))
        self.s, self.conv = up(rng.normal(0, 0.3, (2 * n, hv, dk, dv)).astype(np.float32)), up(rng.normal(0, 1, (2 * n, taps - 1, self.C)).astype(np.float32))
        self.qkv, self.g, self.beta, self.o = hqlib.DevBuf(T * self.C * 2), hqlib.DevBuf(T * hv * 4), hqlib.DevBuf(T * hv * 4), hqlib.DevBuf(T * hv * dv * 2)
        self.st, self.scan = hqlib.States(hk, hv, dk, dv, taps, 2 * n, self.s, self.conv), hqlib.Scan(n, T)
        self.scan.set(self.st, n_new, np.arange(n), np.arange(n, 2 * n), stream=self.stream.ptr)
        self.off, self.gated, self.dk = (2 * hk * dk, 4 * hk * dk), gated, dk
        self.k, self.v = (up(rng.normal(0, 1, (6, 16, 2, 64)).astype(np.float16)) for _ in range(2))
        self.kv = hqlib.KvCache(hqlib.KV_F16, 6, 16, 2, 64, self.k, self.v, (16 * 2 * 64, 2 * 64, 64))
        self.V, self.B = 20011, 4
        self.logits, self.score = up(rng.normal(0, 3, (2 * self.B, self.V)).astype(np.float32)), up(rng.normal(0, 1, 2 * self.B).astype(np.float32))
        self.out = [hqlib.DevBuf(2 * 8 * 4) for _ in range(3)]

    def run(self):
        h, p = self.hq, self.stream.ptr
        h.delta_append(self.scan, self.st, self.x, self.w, self.a, self.b, self.al, self.dt, self.qkv, self.g, self.beta, f32=True, stream=p)
        kw = dict(norm=self.norm, gate=self.z) if self.gated else {}
        h.delta(self.scan, self.st, self.qkv, self.qkv.ptr + self.off[0], self.qkv.ptr + self.off[1], self.g, self.beta, self.o, self.dk ** -0.5,
                qk_stride=self.C, v_stride=self.C, stream=p, **kw)
        h.kv_copy([self.kv], [0, 1], [4, 5], [16, 7], stream=p)
        h.beam(self.logits, 2, self.B, self.V, self.score, 8, *self.out, f32=True, stream=p)

    def results(self):
        return [d.download((d.nbytes,), np.uint8) for d in (self.qkv, self.g, self.beta, self.o, self.s, self.conv, self.k, self.v, *self.out)]

    def clear(self):
        for d in (self.qkv, self.g, self.beta, self.o, *self.out):
            d.upload(np.full(d.nbytes, 0xa5, np.uint8))


def same(a, b):
    return all(np.array_equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("n_new,gated", [([1500, 1, 70, 5, 0], True), ([1, 1, 3], False)])
def test_captured_step(hqlib, hip, n_new, gated):
    print(f"[gpu] captured step {n_new}", flush=True)
    step = Step(hqlib, 3, n_new, gated)
    step.run()  # (workspaces of this stream grow here)
    step.stream.sync()
    want = step.results()
    graph, run = C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(C.c_void_p(step.stream.ptr), 1) == 0
    step.run()
    assert hip.hipStreamEndCapture(C.c_void_p(step.stream.ptr), C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
    for i in range(4):
        step.clear()
        hqlib.synchronize()
        assert hip.hipGraphLaunch(run, C.c_void_p(step.stream.ptr)) == 0
        step.stream.sync()
        assert same(step.results(), want), f"replay {i}"
        step.run()  # eager work between the replays
        step.stream.sync()
        assert same(step.results(), want)
    assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0
    step.scan.free()
    step.stream.destroy()


def test_steps_side_by_side(hqlib):
    """Two steps queued on two streams with no wait between them, each with a description of its own, give what each gives alone."""
    print("[gpu] two steps side by side", flush=True)
    steps = [Step(hqlib, 5, [900, 3, 40], True), Step(hqlib, 6, [2, 1200, 1], False)]
    want = []
    for s in steps:
        s.run()
        s.stream.sync()
        want.append(s.results())
    for _ in range(3):
        for s in steps:
            s.clear()
        hqlib.synchronize()
        for _ in range(4):
            for s in steps:
                s.run()
        for s in steps:
            s.stream.sync()
        assert all(same(s.results(), w) for s, w in zip(steps, want))
    for s in steps:
        s.scan.free()
        s.stream.destroy()
