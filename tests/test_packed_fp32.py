"""No kernel of the library contains a packed fp32 instruction (v_pk_add / mul / fma_f32): some of their forms have given wrong results on these
machines, and -O3 forms them from ordinary float code.  Built for gfx950 without a GPU."""
import concurrent.futures
import glob
import os
import re
import subprocess

import pytest

HIPCC = "/opt/rocm/bin/hipcc"
CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "neural_invertible_warp_amd", "csrc")


def compile_lines():
    """the compiler lines of a whole build, as make would run them"""
    out = subprocess.run(["make", "-C", CSRC, "-n", "-B"], check=True, capture_output=True, text=True).stdout
    return {m[1]: line.split() for line in out.splitlines() if (m := re.search(r" -c (\w+\.hip) ", line))}


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc (cross-compiles gfx950 without a GPU)")
def test_no_kernel_has_a_packed_fp32_instruction(tmp_path):
    lines = compile_lines()
    assert sorted(lines) == sorted(os.path.basename(p) for p in glob.glob(os.path.join(CSRC, "*.hip")))

    def packed(name):
        cmd = lines[name]
        out = str(tmp_path / (name + ".s"))
        cmd = cmd[:cmd.index("-c")] + ["-S", "--cuda-device-only", name, "-o", out]
        subprocess.run(cmd, check=True, cwd=CSRC, capture_output=True, timeout=600)
        return name, sorted(set(re.findall(r"v_pk_(?:add|mul|fma)_f32", open(out).read())))

    with concurrent.futures.ThreadPoolExecutor(max_workers=4) as pool:
        found = {name: ops for name, ops in pool.map(packed, sorted(lines)) if ops}
    assert not found, found
