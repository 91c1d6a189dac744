"""The same hazard as test_lds_dma_hazard.py along every way that control can take to a DMA: through a label that is fallen
into, round a loop's back edge, over a taken branch.  A block's history there is the tail of every block before it.
CPU-only: hipcc cross-compiles for gfx950."""
import concurrent.futures as cf
import re
import subprocess

from aubier_amd import build as B

from test_lds_dma_hazard import WAIT_STATES, pytestmark, scalar_registers  # noqa: F401

# vector instructions whose second operand is a scalar result as well (carries, division's scale)
TWO_RESULTS = re.compile(r"v_(add|sub|subrev|addc|subb|subbrev)_co|v_div_scale|v_mad_[ui]64")
ENDS = ("s_branch", "s_endpgm", "s_setpc_b64", "s_trap")


def registers(text):
    """scalar_registers, with vcc as the registers that it is (106, 107)"""
    out = scalar_registers(text)
    if re.search(r"\bvcc(_lo)?\b", text):
        out.add(106)
    if re.search(r"\bvcc(_hi)?\b", text):
        out.add(107)
    return out


def written(op, args):
    """The scalar registers that a vector instruction writes"""
    if not op.startswith("v_"):
        return set()
    dst = re.split(r",\s*", args)
    out = registers(dst[0])
    if TWO_RESULTS.match(op) and len(dst) > 1:
        out |= registers(dst[1])
    if op.startswith("v_cmp") and not op.startswith("v_cmpx") and op.endswith("_e32"):
        out |= {106, 107}
    return out


def read(listing):
    """([(line, op, args)], {index of an instruction: the instructions that may run right before it})"""
    code, before, labels, pending = [], {}, {}, []
    for n, line in enumerate(listing.splitlines(), 1):
        line = line.split(";")[0].split("//")[0].strip()
        if not line or (line.startswith(".") and not line.endswith(":")):
            continue
        if line.endswith(":"):
            labels[line[:-1]] = len(code)
            continue
        op, _, args = line.partition(" ")
        args = args.strip()
        i = len(code)
        code.append((n, op, args))
        before.setdefault(i, [])
        if i and not code[i - 1][1].startswith(ENDS):
            before[i].append(i - 1)
        if op == "s_branch" or op.startswith("s_cbranch"):
            pending.append((i, args))
    for i, to in pending:
        if to in labels and labels[to] < len(code):
            before[labels[to]].append(i)
    return code, before


def hazards(listing):
    """(DMA instructions, [(line, writer's line, writer, its registers, wait states between)])"""
    code, before = read(listing)
    seen, found = 0, set()
    for i, (line, op, args) in enumerate(code):
        if not (re.match(r"(buffer|global)_load", op) and re.search(r"\blds\b|_lds_", op + " " + args)):
            continue
        seen += 1
        need = registers(args) | {"m0"}
        # (instruction, registers still of interest, wait states from behind it to the DMA), fewest states first
        todo, least = [(p, need, 0) for p in before[i]], {}
        while todo:
            at, regs, states = todo.pop()
            if states >= WAIT_STATES or least.get((at, frozenset(regs)), WAIT_STATES) <= states:
                continue
            least[at, frozenset(regs)] = states
            n, o, a = code[at]
            hit = written(o, a) & regs
            if hit:
                found.add((line, n, o, tuple(sorted(map(str, hit))), states))
            if o.startswith(("s_", "v_")) and not o.startswith(("s_cmp", "s_nop", "s_cbranch", "s_bitcmp", "s_waitcnt", "s_barrier")):
                # (a register that is written anew since is no longer the vector instruction's)
                regs = regs - registers(re.split(r",\s*", a)[0]) if a else regs
            if regs:
                todo += [(p, regs, states + (int(a, 0) + 1 if o == "s_nop" else 1)) for p in before[at]]
    return seen, sorted(found)


DMA = "buffer_load_dwordx4 v1, s[8:11], s4 offen lds"


def test_the_reader_follows_control():
    load = f"s_mov_b32 m0, s2\ns_nop 0\n{DMA}\n"
    def finds(text):
        return bool(hazards(text)[1])
    assert finds(f"v_readlane_b32 s9, v255, 3\n{load}")
    assert finds(f"v_readlane_b32 s9, v255, 3\n.LBB0_1:\n{load}")                                   # a label that is fallen into
    assert finds(f"s_branch .LBB0_2\n.LBB0_1:\n{load}s_endpgm\n.LBB0_2:\nv_readfirstlane_b32 s8, v0\ns_branch .LBB0_1\n")     # a branch to it
    assert finds(f".LBB0_1:\n{load}v_readlane_b32 s4, v255, 3\ns_cbranch_scc1 .LBB0_1\ns_endpgm\n")  # a loop's back edge
    assert finds(f"v_mov_b32 v0, v1\nv_add_co_u32 v0, s[10:11], v0, v1\n{load}")                     # a carry
    assert not finds(f"v_readlane_b32 s9, v255, 3\ns_nop 3\n.LBB0_1:\n{load}")                       # far enough
    assert not finds(f"v_readlane_b32 s9, v255, 3\ns_branch .LBB0_9\n.LBB0_1:\n{load}s_endpgm\n.LBB0_9:\ns_endpgm\n")     # control never gets there
    assert not finds(f"v_readlane_b32 s9, v255, 3\ns_mov_b32 s9, s20\n{load}")                       # written anew
    assert not finds(f"v_readlane_b32 s19, v255, 3\n{load}")


def test_no_way_to_a_dma_writes_its_registers_too_late():
    srcs = sorted(B.CSRC.glob("*.hip"))

    def listing(src):
        r = subprocess.run([B.HIPCC, *B.HIP_FLAGS, "-I", str(B.ROOT / "include"), "--offload-device-only", "-S", str(src), "-o", "-"],
                           stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)
        assert r.returncode == 0, r.stderr[-2000:]
        return hazards(r.stdout)

    with cf.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        got = dict(zip(srcs, ex.map(listing, srcs)))
    assert sum(seen for seen, _ in got.values()) > 500
    for src, (seen, found) in got.items():
        assert not found, (src.name, len(found), found[:5])
