"""The compiled products (CPU only): M0 belongs to the copies into LDS, every copy is counted by a wait, and no tile's sums spill."""
import os
import re
import subprocess

import pytest

import test_asm_invariants as inv


@pytest.fixture(scope="module", params=["linear", "linear_grad"])
def lines(request, tmp_path_factory):
    b = inv._build_module()
    if not os.path.exists(b.HIPCC):
        pytest.skip("hipcc is not installed")
    out = tmp_path_factory.mktemp("asm") / f"{request.param}.s"
    flags = [f for f in b.CFLAGS if f != "-fPIC"]
    r = subprocess.run([b.HIPCC, *flags, "-I", b.CSRC, "--cuda-device-only", "-S", os.path.join(b.CSRC, f"{request.param}.hip"),
                        "-o", str(out)], capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stderr[-2000:]
    return out.read_text().splitlines()


def test_m0_belongs_to_the_copies(lines):
    asm = [s for s in (l.split(";")[0].strip() for l in lines) if s and not s.startswith(".")]
    uses = [i for i, l in enumerate(asm) if re.search(r"\bm0\b", l)]
    assert uses
    for i in uses:
        assert re.match(r"s_mov_b32 m0, (s\d+|vcc_lo|vcc_hi|ttmp\d+)$", asm[i]), asm[i]
        assert asm[i + 1] == "s_nop 0", asm[i + 1]
        assert re.match(r"buffer_load_dwordx4 v\d+, s\[\d+:\d+\], 0 offen lds$", asm[i + 2]), asm[i + 2]
    assert len(uses) == len([l for l in asm if re.search(r"\blds$", l)])
    other = re.compile(r"^(s_movrel|v_movrel|s_set_gpr_idx|s_sendmsg|ds_gws|v_interp|s_ttracedata|ds_append|ds_consume)")
    assert not [l for l in asm if other.match(l)]


def test_nothing_spills(lines):
    sizes = [int(m.group(1)) for l in lines if (m := re.search(r"\.private_segment_fixed_size:\s+(\d+)", l))]
    assert len(sizes) >= 10 and not any(sizes)
