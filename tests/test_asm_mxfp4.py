"""The compiled MXFP4 experts (CPU only): M0 belongs to the LDS copies, and the several-pass
conversions to and from E2M3 never write over their own operands."""
import os
import re
import subprocess

import pytest

import test_asm_invariants as inv


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    b = inv._build_module()
    if not os.path.exists(b.HIPCC):
        pytest.skip("hipcc is not installed")
    out = tmp_path_factory.mktemp("asm") / "mxfp4_experts.s"
    flags = [f for f in b.CFLAGS if f != "-fPIC"]
    r = subprocess.run([b.HIPCC, *flags, "-I", b.CSRC, "--cuda-device-only", "-S",
                        os.path.join(b.CSRC, "mxfp4_experts.hip"), "-o", str(out)], capture_output=True, text=True,
                       timeout=900)
    assert r.returncode == 0, r.stderr[-2000:]
    lines = [l.split(";")[0].strip() for l in out.read_text().splitlines()]
    return [l for l in lines if l and not l.startswith(".")]


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
