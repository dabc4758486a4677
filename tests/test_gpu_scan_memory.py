"""Device memory of hq_scan: what a step's passes need one after another they share."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu


def free_bytes(hqlib):
    a, b = C.c_size_t(), C.c_size_t()
    hqlib.synchronize()
    assert hqlib.load().hipMemGetInfo(C.byref(a), C.byref(b)) == 0
    return a.value


def used(hqlib, n, hk, hv, d):
    before = free_bytes(hqlib)
    scan = hqlib.Scan(1, n)
    scan.set(hqlib.States(hk, hv, d, d, 4, 1, None, None), [n], [0], [0])
    now = before - free_bytes(hqlib)
    scan.free()
    return now


def test_places_of_parts(hqlib):
    """One sequence in parts over 40 and over 320 passes: the states between parts have their places in every pass anew, and the longer
    step only has longer lists (12 bytes for 8 tokens, 8 for 64 and some for each part, with half of that as room: below 3 bytes a
    token; 2 MiB rounding of each of three allocations)."""
    print("[gpu] memory of long steps", flush=True)
    few, many = (used(hqlib, n, 16, 32, 128) for n in (1 << 20, 1 << 23))
    assert few > 0 and many - few <= 3 * ((1 << 23) - (1 << 20)) + 3 * (2 << 20)


def test_memory_is_kept_for_steps_and_returned(hqlib):
    """A step that fits what an earlier one had allocates nothing, and hq_scan_free gives everything back."""
    print("[gpu] memory of steps in a row", flush=True)
    used(hqlib, 4096, 2, 4, 64)
    before = free_bytes(hqlib)
    scan = hqlib.Scan(8, 1 << 16)
    st = hqlib.States(2, 4, 64, 64, 4, 16, None, None)
    scan.set(st, [1 << 15, 1 << 14], [0, 1], [2, 3])
    most = free_bytes(hqlib)
    for n in ([100, 7, 2000], [1] * 8, [1 << 14], [1 << 15, 1 << 14], [0]):
        scan.set(st, n, list(range(len(n))), list(range(len(n))))
        assert free_bytes(hqlib) == most
    scan.free()
    assert free_bytes(hqlib) >= before
