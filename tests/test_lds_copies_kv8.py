"""The 8-bit attention kernels' copies from global memory to LDS, in the assembly
hipcc makes of them: m0 is written right before each with the wait state that
asks for, and a scalar base is one that the scalar unit wrote."""
import os
import re
import shutil
import subprocess

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flashengine.cpp_amd")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no HIP compiler")
def test_copies_have_their_wait_states(tmp_path):
    out = tmp_path / "attn.s"
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-mcode-object-version=5", "-Xclang",
                    "-target-feature", "-Xclang", "-packed-fp32-ops", "-I" + os.path.join(PKG, "..", "include"),
                    "-I" + os.path.join(PKG, "csrc"), "--cuda-device-only", "-S",
                    os.path.join(PKG, "csrc", "attn_kv8.hip"), "-o", str(out)],
                   check=True, timeout=300, stderr=subprocess.DEVNULL)
    before = ["", ""]
    wide = narrow = 0
    for line in out.read_text().splitlines():
        line = line.split(";")[0].strip()
        if not line or line.endswith(":") or line.startswith("."):
            continue
        m = re.match(r"global_load_lds_dword(x4)? v\S+, (off|s\[\d+:\d+\])", line)
        if m:
            wide, narrow = wide + (m[1] is not None), narrow + (m[1] is None)
            assert re.match(r"s_mov_b32 m0, (s\d+|vcc_lo|vcc_hi)$", before[0]), (before, line)
            if m[2] == "off":
                assert before[1] == "s_nop 0", (before, line)
            else:
                assert before[1].startswith(("s_mov_b64 " + m[2] + ", s[", "s_mov_b64 " + m[2] + ", vcc")), (before, line)
        before = [before[1], line]
    assert wide > 300 and narrow > 50
