"""hq.py's ctypes mirrors of the recurrent layers' structs have the offsets of include/hq_serve.h."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

import hq

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_mirrors_match_the_header(tmp_path):
    if not shutil.which("gcc"):
        pytest.skip("gcc not found")
    structs = {"hq_kv_t": hq.Kv, "hq_state_t": hq.State, "hq_delta_in_t": hq.DeltaIn, "hq_delta_t": hq.Delta}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "hq_serve.h"', "int main(void) {"]
    want = []
    for name, cls in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append((name, C.sizeof(cls)))
        for f, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {f}));')
            want.append((f"{name}.{f}", getattr(cls, f).offset))
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text("\n".join(lines + ["return 0; }"]) + "\n")
    subprocess.run(["gcc", "-std=c11", f"-I{os.path.join(ROOT, 'include')}", str(src), "-o", str(exe)], check=True)
    got = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()
    assert [(n, int(g)) for (n, _), g in zip(want, got)] == want and len(got) == len(want)
