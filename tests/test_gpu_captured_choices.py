"""hq_beam and hq_logprobs captured into graphs, beside calls of larger shapes on the same stream: a graph goes on with the workspace that it was
captured with. (Memory that the larger calls could have given back is taken and filled before each replay.)"""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip(hqlib):
    L = hqlib.load()  # (its dependencies' functions are found through it)
    for f in ("hipStreamBeginCapture", "hipStreamEndCapture", "hipGraphInstantiate", "hipGraphLaunch", "hipGraphDestroy", "hipGraphExecDestroy", "hipMemGetInfo"):
        getattr(L, f).restype = C.c_int
    return L


class Call:
    def __init__(self, hqlib, stream, seed, G, B, V, k):
        rng = np.random.default_rng(seed)
        self.hq, self.stream, self.shape, self.k = hqlib, stream, (G, B, V), k
        self.x, self.score = hqlib.DevBuf.from_array(rng.normal(0, 3, (G * B, V)).astype(np.float16)), hqlib.DevBuf.from_array(rng.normal(-9, 3, G * B).astype(np.float32))
        self.out = [hqlib.DevBuf(G * k * 4) for _ in range(3)] + [hqlib.DevBuf(G * B * 4), hqlib.DevBuf(G * B * k * 4), hqlib.DevBuf(G * B * k * 4)]

    def run(self):
        G, B, V = self.shape
        self.hq.beam(self.x, G, B, V, self.score, self.k, *self.out[:3], f32=False, stream=self.stream.ptr)
        self.hq.logprobs(self.x, G * B, V, f32=False, top_k=self.k, entropy=self.out[3], top_ids=self.out[4], top_logp=self.out[5], stream=self.stream.ptr)

    def results(self):
        self.stream.sync()
        return [b.download((b.nbytes,), np.uint8) for b in self.out]

    def clear(self):
        for b in self.out:
            b.upload(np.full(b.nbytes, 0xa5, np.uint8))


SHAPES = [(1, 4, 32000, 4), (2, 8, 151936, 16), (16, 8, 20000, 8), (100, 8, 3000, 64), (700, 4, 400, 3)]


def test_graphs_beside_larger_calls(hqlib, hip):
    stream = hqlib.Stream()
    calls, graphs, want = [], [], []
    for i, shape in enumerate(SHAPES):
        print(f"[gpu] captured choices {shape}", flush=True)
        c = Call(hqlib, stream, i, *shape)
        c.run()  # (workspaces grow here, past those of the graphs before)
        want.append(c.results())
        graph, run = C.c_void_p(), C.c_void_p()
        assert hip.hipStreamBeginCapture(C.c_void_p(stream.ptr), 1) == 0
        c.run()
        assert hip.hipStreamEndCapture(C.c_void_p(stream.ptr), C.byref(graph)) == 0
        assert hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
        calls.append(c), graphs.append((graph, run))
        taken = [hqlib.DevBuf.from_array(np.full(n, 0xff, np.uint8)) for n in (1 << 12, 1 << 13, 1 << 14, 1 << 16, 1 << 18, 1 << 20, 1 << 21) for _ in range(4)]
        for _ in range(2):
            for j, (_, g) in enumerate(graphs):
                calls[j].clear()
                hqlib.synchronize()
                assert hip.hipGraphLaunch(g, C.c_void_p(stream.ptr)) == 0
                assert all(np.array_equal(a, b) for a, b in zip(calls[j].results(), want[j])), (i, j)
                c.run()  # eager work between the replays
                assert all(np.array_equal(a, b) for a, b in zip(c.results(), want[i])), (i, j)
        assert all((t.download((t.nbytes,), np.uint8) == 0xff).all() for t in taken)
        del taken
    for graph, run in graphs:
        assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0
    stream.destroy()


def test_a_stream_gives_its_workspaces_back(hqlib, hip):
    def free():
        a, b = C.c_size_t(), C.c_size_t()
        hqlib.synchronize()
        assert hip.hipMemGetInfo(C.byref(a), C.byref(b)) == 0
        return a.value

    def work():
        stream = hqlib.Stream()
        rows, score, out = hqlib.DevBuf.from_array(np.zeros(1 << 20, np.float32)), hqlib.DevBuf.from_array(np.zeros(1 << 20, np.float32)), [hqlib.DevBuf(1 << 25) for _ in range(3)]
        for n in (1, 1000, 100000, 1 << 20):
            hqlib.beam(rows, n, 1, 1, score, 8, *out, f32=True, stream=stream.ptr)
        stream.sync()
        stream.destroy()
    print("[gpu] workspaces of streams", flush=True)
    work()
    before = free()
    for _ in range(3):
        work()
    assert free() >= before - (2 << 20)
