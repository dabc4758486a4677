"""hip_batch_step that fails behind its first kernels (include/hq_backend.h: synchronous): it returns with nothing under way,
since what it queued reads the host array that the next step writes."""
import time

import numpy as np
import pytest

from test_gpu_backend_options import Q8, make

pytestmark = pytest.mark.gpu


def test_nothing_is_under_way_behind_a_failed_step(hqlib):
    model = make(3, Q8, False, True, 0.0, 32, 4, 128, 128)
    model["cfg"]["eps"] = -1.0  # what the first layer's append refuses, behind the embedding and the first product
    be = hqlib.HipBackend(hqlib.RefModelView(model), 64)
    n = 60000
    s = hqlib.HipBatch(be, n // 64 + 1, 64, 1, n, n // 64 + 1)
    tokens, pages = np.arange(n) % 512, np.arange(n // 64 + 1)[None]
    print("[gpu] failing steps", flush=True)
    calls, waits = [], []
    for _ in range(4):
        t0 = time.perf_counter()
        with pytest.raises(hqlib.HQError, match="eps"):
            s.step(tokens, [n], [n], pages, top_k=1)
        t1 = time.perf_counter()
        hqlib.synchronize()
        calls.append(t1 - t0), waits.append(time.perf_counter() - t1)
        print(f"[gpu]   step {calls[-1] * 1e3:.2f} ms, waited {waits[-1] * 1e3:.3f} ms", flush=True)
    assert min(waits) < 0.25 * min(calls)
    s.free()
    be.destroy()
