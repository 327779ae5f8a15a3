"""csrc/niw_optim.hip takes tensors that are aligned to their own element and no more (a view may begin anywhere in a buffer): what it promises the
compiler about its vector accesses, read from the intermediate code of a build for gfx950 (no GPU)."""
import os
import re
import subprocess

import pytest

HIPCC = "/opt/rocm/bin/hipcc"
CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "neural_invertible_warp_amd", "csrc")
BYTES = {"float": 4, "i32": 4, "i16": 2, "i64": 8}


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc (cross-compiles gfx950 without a GPU)")
def test_vector_accesses_promise_no_more_than_an_element(tmp_path):
    out = str(tmp_path / "optim.ll")
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-I", os.path.join(CSRC, "..", "..", "include"), "-I", CSRC, "--cuda-device-only", "-S",
                    "-emit-llvm", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", os.path.join(CSRC, "niw_optim.hip"), "-o", out], check=True,
                   capture_output=True, timeout=300)
    kernel, seen, promised = None, 0, []
    for line in open(out):
        m = re.match(r"define .*?@(\w+)\(", line)
        kernel = m[1] if m else kernel
        # (what is read of a table's slots or through the kernel arguments is aligned by construction: other address spaces and scalar types)
        m = re.search(r"(load|store) <(\d+) x (float|i16|i32)>.*?ptr (?!addrspace).*?align (\d+)", line)
        if m and "store_kernel" not in kernel:
            seen += 1
            if int(m[4]) > 4:
                promised.append((kernel, line.strip()))
    assert seen > 500 and not promised, promised[:3]
