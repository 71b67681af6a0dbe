"""The compiled MXFP4 experts (CPU only): M0 belongs to the LDS copies, the tiles' counted waits
cover the copies they are for, and the several-pass conversions to and from E2M3 never write
over their own operands."""
import os
import re
import subprocess

import pytest

import test_asm_invariants as inv


@pytest.fixture(scope="module")
def text(tmp_path_factory):
    b = inv._build_module()
    if not os.path.exists(b.HIPCC):
        pytest.skip("hipcc is not installed")
    out = tmp_path_factory.mktemp("asm") / "mxfp4_experts.s"
    flags = [f for f in b.CFLAGS if f != "-fPIC"]
    r = subprocess.run([b.HIPCC, *flags, "-I", b.CSRC, "--cuda-device-only", "-S",
                        os.path.join(b.CSRC, "mxfp4_experts.hip"), "-o", str(out)], capture_output=True, text=True,
                       timeout=900)
    assert r.returncode == 0, r.stderr[-2000:]
    return [l.split(";")[0].strip() for l in out.read_text().splitlines()]


@pytest.fixture(scope="module")
def asm(text):
    return [l for l in text if l and not l.startswith(".")]


def test_m0_belongs_to_the_lds_copies(asm):
    uses = [i for i, l in enumerate(asm) if re.search(r"\bm0\b", l)]
    assert uses
    for i in uses:
        assert re.match(r"s_mov_b32 m0, (s\d+|vcc_lo|vcc_hi|ttmp\d+)$", asm[i]), asm[i]
        assert asm[i + 1] == "s_nop 0", asm[i + 1]
        assert asm[i + 2].startswith("global_load_lds_dword"), asm[i + 2]
    assert len(uses) == len([l for l in asm if l.startswith("global_load_lds")])
    inv.test_no_instruction_reads_m0_implicitly(asm)


def _regs(operand: str) -> set:
    m = re.match(r"v\[(\d+):(\d+)\]$|v(\d+)$", operand)
    if not m:
        return set()
    lo = int(m.group(1) or m.group(3))
    return set(range(lo, int(m.group(2) or lo) + 1))


def test_conversions_do_not_overwrite_their_operands(asm):
    seen = 0
    for l in asm:
        if re.match(r"v_cvt_scalef32_(2xpk16|pk32)_", l):
            dst, *src = [o.strip() for o in l.split(None, 1)[1].split(", ")]
            for o in src:
                assert not _regs(dst) & _regs(o), l
            seen += 1
    assert seen > 10


def test_nothing_spills(asm):
    assert not [l for l in asm if l.startswith("scratch_")]


def _blocks(text, kernel):
    """{label: (instructions, successors)} of a kernel's basic blocks, and the first label."""
    start = next(i for i, l in enumerate(text) if re.match(rf"_Z\w*{kernel}\w*:", l))
    end = next(i for i in range(start, len(text)) if text[i].startswith(".Lfunc_end"))
    blocks, order, label, n = {"entry": []}, ["entry"], "entry", 0
    for l in text[start + 1:end]:
        m = re.match(r"(\.LBB\w+):", l)
        if m:
            label = m.group(1)
        elif l and not l.startswith("."):
            blocks.setdefault(label, []).append(l)
            if re.match(r"s_c?branch", l):     # what follows a branch is a block of its own
                n += 1
                label = f"after{n}"
            else:
                continue
        else:
            continue
        order.append(label)
        blocks.setdefault(label, [])
    out = {}
    for i, b in enumerate(order):
        ends = blocks[b][-1] if blocks[b] else ""
        to = [ends.split()[1]] if re.match(r"s_c?branch", ends) else []
        if not re.match(r"s_branch|s_endpgm", ends) and i + 1 < len(order):
            to.append(order[i + 1])
        out[b] = (blocks[b], to)
    return out


@pytest.mark.parametrize("kernel,copies", [("tile_gateup_kernelILi2ELi4ELi5E", 3), ("tile_gateup_kernelILi2ELi5ELi5E", 4),
                                           ("tile_down_kernelILi2ELi5E", 4)])
def test_counted_waits_cover_their_copies(text, kernel, copies):
    """Along every path to a barrier behind a wait that lets N loads be under way, at least N loads follow the
    copies of the chunk that is read next: the newest copies in tiles of 64 rows, in those of 32 (`copies` a
    chunk) the ones before the two newest chunks."""
    blocks = _blocks(text, kernel)
    keep = 64                                   # a path's state: its newest loads, c a copy, l another
    state = {b: set() for b in blocks}
    state["entry"] = {""}
    work, waits = ["entry"], {}
    while work:
        b = work.pop()
        cur = set(state[b])
        body, to = blocks[b]
        for i, l in enumerate(body):
            if l.startswith(("global_load", "global_store", "scratch_")):
                op = "c" if l.startswith("global_load_lds") else "l"
                cur = {(s + op)[-keep:] for s in cur}
            m = re.match(r"s_waitcnt vmcnt\((\d+)\) lgkmcnt\(0\)$", l)
            if m and int(m.group(1)) and body[i + 1:i + 2] == ["s_barrier"]:
                waits.setdefault(int(m.group(1)), set()).update(cur)
        for t in to:
            if not cur <= state[t]:
                state[t] |= cur
                work.append(t)
    steady = 4 + 2 * (copies + 4)
    assert set(waits) == {4, 2 * copies, 2 * copies + 4, 2 * copies + 8, steady}
    for n, paths in waits.items():
        newer = 0 if n == 4 else 2 * copies
        for s in paths:
            at = [i for i, op in enumerate(s) if op == "c"]
            assert len(at) > newer and len(s) - 1 - at[-1 - newer] >= n, (n, s)
