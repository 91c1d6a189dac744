"""The LDS DMA is inline assembly, which the compiler's hazard recogniser does not look into: a vector-memory instruction
needs five wait states behind a vector instruction that writes one of its scalar registers (a v_readlane that restores
a spilled buffer resource, a v_readfirstlane, a compare).  With fewer it goes to the address that the registers held
before.  This reads the listing of every kernel built here.  CPU-only: hipcc cross-compiles for gfx950."""
import concurrent.futures as cf
import os
import re
import shutil
import subprocess

import pytest

from aubier_amd import build as B

pytestmark = pytest.mark.skipif(shutil.which(B.HIPCC) is None and not os.path.exists(B.HIPCC), reason="hipcc not available")
WAIT_STATES = 5


def scalar_registers(text):
    out = set()
    for m in re.finditer(r"\bs\[(\d+):(\d+)\]", text):
        out |= set(range(int(m[1]), int(m[2]) + 1))
    out |= {int(m[1]) for m in re.finditer(r"\bs(\d+)\b", text)}
    if re.search(r"\bm0\b", text):
        out.add("m0")
    return out


def hazards(listing):
    """(DMA instructions, [(line, writer, its registers, wait states between)])"""
    seen, found, past = 0, [], []                            # past: (op, registers written by the VALU, wait states)
    for n, line in enumerate(listing.splitlines(), 1):
        line = line.split(";")[0].strip()
        if not line or line.startswith("."):
            continue
        if line.endswith(":"):
            past = []
            continue
        op, _, args = line.partition(" ")
        if re.match(r"(buffer|global)_load", op) and re.search(r"\blds\b|_lds_", line):
            seen += 1
            need, between = scalar_registers(args) | {"m0"}, 0
            for o, regs, states in reversed(past):
                if between >= WAIT_STATES:
                    break
                if regs & need:
                    found.append((n, o, sorted(map(str, regs & need)), between))
                between += states
        written = set()
        if re.match(r"v_(readlane|readfirstlane|cmp)", op):
            written = scalar_registers(args.split(",")[0])
        past = past[-12:] + [(op, written, int(args, 0) + 1 if op == "s_nop" else 1)]
    return seen, found


def test_the_reader_finds_a_planted_one():
    text = "v_readlane_b32 s9, v255, 3\ns_mov_b32 m0, s2\ns_nop 0\nbuffer_load_dwordx4 v1, s[8:11], s4 offen lds\n"
    assert hazards(text)[1] and not hazards(text.replace("s_nop 0", "s_nop 4"))[1]
    assert not hazards(text.replace("s9", "s19"))[1]


def test_no_dma_follows_a_write_of_its_registers_too_closely():
    srcs = [s for s in sorted(B.CSRC.glob("*.hip"))]

    def listing(src):
        r = subprocess.run([B.HIPCC, *B.HIP_FLAGS, "-I", str(B.ROOT / "include"), "--offload-device-only", "-S", str(src), "-o", "-"],
                           stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)
        assert r.returncode == 0, r.stderr[-2000:]
        return hazards(r.stdout)

    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        got = dict(zip(srcs, ex.map(listing, srcs)))
    assert sum(seen for seen, _ in got.values()) > 500
    for src, (seen, found) in got.items():
        assert not found, (src.name, found[:5])
