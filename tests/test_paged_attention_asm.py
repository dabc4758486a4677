"""Device assembly scan (CPU, no GPU): no k_rows kernel of the paged attention uses scratch memory.

Its tiles come by LDS DMA that the compiler does not track, and waits count the loads behind the one that is needed
(s_waitcnt vmcnt(n)). Scratch loads and stores are counted too: a kernel that spills would read tiles before they are there."""
import os
import re
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "..", "hilbert-pruned-8b_amd", "csrc")
ASM = os.path.abspath(os.path.join(HERE, "..", "hilbert-pruned-8b_amd", "_build", "asm", "hq_paged_attention.s"))


def kernels(text, name):
    """(symbol, body) of every kernel whose name holds `name`."""
    return re.findall(r"^(_Z\w*%s\w*):.*?\n(.*?)^\s*\.end_amdhsa_kernel" % name, text, re.M | re.S)


def spills(body):
    return len(re.findall(r"^\s*(?:scratch_\w+|buffer_(?:load|store)\w* .*\bs32\b)", body, re.M))


def test_scanner():
    text = "_ZN1k_rowsE: ; @x\n\tscratch_store_dword off, v1, s32\n\t.end_amdhsa_kernel\n_ZN1k_joinE:\n\ts_endpgm\n\t.end_amdhsa_kernel\n"
    assert [spills(b) for _, b in kernels(text, "k_rows")] == [1] and [spills(b) for _, b in kernels(text, "k_join")] == [0]


@pytest.mark.timeout(900)
def test_rows_kernels_do_not_spill():
    subprocess.run(["make", "-s", "-C", CSRC, ASM], check=True, capture_output=True)
    found = kernels(open(ASM).read(), "k_rows")
    assert len(found) == 16, [n for n, _ in found]
    assert not {n: spills(b) for n, b in found if spills(b)}
