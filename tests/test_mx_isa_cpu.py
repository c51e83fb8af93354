"""Static invariants of the block-scaled operators' code objects (no GPU): no spills, no waterfall loops, and no instruction between an
LDS read written in inline assembly and the wait behind it that touches the registers the read will fill -- the compiler takes them
as written at once and may move or reuse them."""
import os
import re
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tools"))

import isa_audit  # noqa: E402

OBJECTS = ("mx.hip.o", "mx_gemm.hip.o", "mx_wgrad.hip.o")


def _object(name):
    path = os.path.join(isa_audit.BUILD, name)
    if not os.path.exists(path):
        pytest.skip("objects not built (make -C latent-diffusion_amd/csrc)")
    return path


@pytest.mark.parametrize("name", OBJECTS)
def test_no_spills_and_no_waterfall_loops(name, tmp_path):
    rows = isa_audit.audit(_object(name), str(tmp_path))
    assert rows
    for r in rows:
        assert r["scratch"] == 0 and r["scratch_ops"] == 0, (r["kernel"], "spills", r["scratch"], r["scratch_ops"])
        assert r["waterfall"] == 0, (r["kernel"], "waterfall loops", r["waterfall"])


def _registers(text):
    out = set()
    for one, lo, hi in re.findall(r"\bv(?:(\d+)|\[(\d+):(\d+)\])", text):
        out.update([int(one)] if one else range(int(lo), int(hi) + 1))
    return out


def pending_read_hazards(listing):
    """(LDS reads seen, instructions that touch a destination of one before a wait for it), along every path through the listing.
    What is carried along: for each register that a read will fill, how many LDS operations have been issued since on the path with the
    fewest (lgkmcnt(n) waits for all that n or more others followed)."""
    code = []
    for line in listing.splitlines():
        ins, _, where = line.partition("//")
        if ins.strip():
            op, _, rest = ins.strip().partition(" ")
            code.append((op, rest.strip(), int(where.split(":")[0], 16) if where.strip() else len(code), _registers(rest)))
    at = {addr: i for i, (_, _, addr, _) in enumerate(code)}
    state, bad, work = {0: {}}, set(), [0]

    def reach(i, pending):
        old = state.get(i)
        new = dict(pending) if old is None else {r: min(old.get(r, 99), pending.get(r, 99)) for r in {*old, *pending}}
        if new != old:
            state[i] = new
            work.append(i)

    while work:
        i = work.pop()
        if i >= len(code):
            continue
        pending = dict(state[i])
        op, rest, addr, regs = code[i]
        if op == "s_waitcnt":
            m = re.search(r"lgkmcnt\((\d+)\)", rest)
            if m:
                pending = {r: n for r, n in pending.items() if n < int(m.group(1))}
        elif regs & pending.keys():
            bad.add(f"{op} {rest}")
        if op.startswith("ds_"):
            pending = {r: min(n + 1, 64) for r, n in pending.items()}
            if op.startswith("ds_read"):
                pending.update(dict.fromkeys(_registers(rest.split(",")[0]), 0))
        if op == "s_branch" or op.startswith("s_cbranch"):
            step = int(rest.split()[0])
            reach(at[addr + 4 + 4 * (step - 65536 if step > 32767 else step)], pending)
        if op not in ("s_branch", "s_endpgm"):
            reach(i + 1, pending)
    return sum(op.startswith("ds_read") for op, _, _, _ in code), sorted(bad)


def test_the_hazard_check_finds_one():
    good = "ds_read_b128 v[4:7], v1 offset:16\nv_add_u32 v2, v1, v1\ns_waitcnt lgkmcnt(0)\nv_add_u32 v2, v4, v1\n"
    assert pending_read_hazards(good) == (1, [])
    early = "ds_read_b128 v[4:7], v1\nds_read_b32 v9, v1\ns_waitcnt lgkmcnt(1)\nv_mov_b32 v2, v7\nv_mov_b32 v3, v9\n"
    assert pending_read_hazards(early) == (2, ["v_mov_b32 v3, v9"])
    # around a loop: the read at its end is under way when the body begins again; the code behind the branch is not on the way
    loop = ("s_nop 0 // 00: x\nv_mov_b32 v2, v9 // 04: x\nds_read_b32 v9, v1 // 08: x\ns_branch 65533 // 0c: x\nv_mov_b32 v3, v9 // 10: x\n")
    assert pending_read_hazards(loop) == (1, ["ds_read_b32 v9, v1", "v_mov_b32 v2, v9"])


@pytest.mark.parametrize("name", ["mx_gemm.hip.o", "mx_wgrad.hip.o"])
def test_nothing_touches_a_register_that_an_lds_read_will_fill(name, tmp_path):
    listing = subprocess.run([isa_audit.LLVM + "/llvm-objdump", "-d", isa_audit.code_object(_object(name), str(tmp_path))], capture_output=True,
                             text=True).stdout
    total = 0
    for m in re.finditer(r"^[0-9a-f]+ <([^>]+)>:\n(.*?)(?=^[0-9a-f]+ <|\Z)", listing, re.S | re.M):
        reads, bad = pending_read_hazards(m.group(2))
        total += reads
        assert not bad, (m.group(1), bad[:5])
    assert total > 100
