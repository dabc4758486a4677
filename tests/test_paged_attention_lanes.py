"""Device assembly scan (CPU, no GPU): what the paged attention's kernels do with all lanes on.

k_rows keeps the pages of 64 tiles in one register, a tile a lane, and takes a tile's with v_readlane. Under a mask that turns
lanes off, the compiler may read a copy of that register which it has just made for the lanes that are on alone: what the lane
asked for holds then is another number, and an address formed from it lies anywhere. Its LDS DMA sets a mask of its own and
turns all lanes on behind it, which would be wrong where some are off."""
import os
import re
import subprocess

import pytest

from test_paged_attention_asm import ASM, CSRC, kernels

def blocks(body):
    """Basic blocks of a kernel: {label: (instructions, labels that may follow)}; the first is ''."""
    out, name, ins, in_asm, n = {}, "", [], False, 0

    def close(after):
        out[name] = (ins, after)

    for line in body.splitlines():
        x = line.split(";")[0].strip()
        if "#ASMSTART" in line or "#ASMEND" in line:
            in_asm = "#ASMSTART" in line
        elif in_asm and "_lds_" in x:
            ins.append("dma")
        label = re.match(r"(\.LBB\w+):", x)
        if label:
            close([label[1]])
            name, ins = label[1], []
        elif x and not in_asm:  # (the LDS DMA's masks are undone within its block)
            ins.append(x)
            jump = re.match(r"s_c?branch\w*\s+(\S+)", x)
            if jump or x == "s_endpgm":
                n += 1
                close(([jump[1]] if jump else []) + ([f"+{n}"] if x.startswith("s_cbranch") else []))
                name, ins = f"+{n}", []
    close([])
    return out


def step(masks, x):
    """The masks that narrow exec, innermost last, behind instruction x."""
    m = re.match(r"s_(and|andn2)_saveexec_b64 (s\[\S+\]|vcc),", x)
    if m:
        return masks + (m[2],)
    m = re.match(r"s_xor_b64 exec, exec, (\S+)", x)
    if m:
        return masks + (m[1],)
    m = re.match(r"s_andn2_b64 exec, exec, (\S+)", x)  # a loop's lanes leave it
    if m:
        return masks if masks[-1:] == ("loop " + m[1],) else masks + ("loop " + m[1],)
    m = re.match(r"s_or_saveexec_b64 (\S+),", x) or re.match(r"s_or_b64 exec, exec, (\S+)", x)
    if m and masks:
        at = [i for i, k in enumerate(masks) if k.split()[-1] == m[1]]  # (spilled and back in others: the innermost)
        return masks[:at[-1]] if at else masks[:-1]
    return () if re.match(r"s_mov_b64 exec, -1", x) else masks


def masked(body):
    """v_readlane instructions and LDS DMA under a mask; but not v_readlane of registers that only v_writelane writes (the
    compiler's store of spilled scalars, which needs no lane to be on)."""
    code = blocks(body)
    others = set()
    for ins, _ in code.values():
        for x in ins:
            d = re.match(r"(?!v_writelane)(?:v|ds|global|buffer|scratch|flat)_\S+\s+v(?:(\d+)|\[(\d+):(\d+)\])", x)
            if d and "store" not in x and "write" not in x:
                others |= {int(d[1])} if d[1] else set(range(int(d[2]), int(d[3]) + 1))
    entry, todo = {"": ()}, [""]
    while todo:
        b = todo.pop()
        masks = entry[b]
        for x in code[b][0]:
            masks = step(masks, x)
        assert len(masks) < 64, "masks that never end: the scan does not know this code"
        for t in code[b][1]:
            if t in code and (t not in entry or len(masks) > len(entry[t])):  # where ways meet, the narrower
                entry[t] = masks
                todo.append(t)
    found = []
    for b, masks in entry.items():
        for x in code[b][0]:
            masks = step(masks, x)
            r = re.match(r"v_readlane_b32 \S+, v(\d+),", x)
            if masks and (x == "dma" or r and int(r[1]) in others):
                found.append(x)
    return found


def test_scanner():
    bad = """v_accvgpr_read_b32 v9, a1
    s_and_saveexec_b64 s[0:1], vcc
    v_readlane_b32 s24, v9, s21
    v_readlane_b32 s25, v255, 3
    s_cbranch_execz .LBB0_1
    v_readlane_b32 s26, v9, 4
    ;;#ASMSTART
    s_mov_b64 exec, s[4:5]
    global_load_lds_dword v[2:3], off
    s_mov_b64 exec, -1
    ;;#ASMEND
    .LBB0_1:
    s_or_b64 exec, exec, s[0:1]
    v_readlane_b32 s24, v9, s21"""
    assert masked(bad) == ["v_readlane_b32 s24, v9, s21", "v_readlane_b32 s26, v9, 4", "dma"]


@pytest.mark.timeout(900)
def test_lanes_are_read_with_all_lanes_on():
    subprocess.run(["make", "-s", "-C", CSRC, ASM], check=True, capture_output=True)
    text = open(ASM).read()
    found = kernels(text, "k_rows") + kernels(text, "k_stream") + kernels(text, "k_join")
    assert len(found) > 16
    assert not {n: masked(b) for n, b in found if masked(b)}
