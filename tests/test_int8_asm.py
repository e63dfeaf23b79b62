"""The LDS copies of the eight-bit product, as built for gfx950: the same
check of their inline assembly as the other kernels' (test_asm_hazards.py).
No GPU needed."""

import os
import shutil
import subprocess

import pytest

from test_asm_hazards import _COPY, HIPCC, KDIR, ROOT, hazards


@pytest.mark.skipif(not shutil.which(HIPCC) and not os.path.exists(HIPCC), reason="hipcc not available")
def test_lds_copies_of_the_int8_product_have_no_sgpr_hazard(tmp_path):
    out = tmp_path / "gemm_int8.s"
    cmd = [HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
           "-packed-fp32-ops", "-I" + os.path.join(ROOT, "include"), "-I" + KDIR, "--cuda-device-only", "-S",
           os.path.join(KDIR, "gemm_int8.hip"), "-o", str(out)]
    subprocess.run(cmd, check=True, capture_output=True, timeout=300)
    asm = out.read_text()
    assert sum(1 for line in asm.splitlines() if _COPY.match(line.strip())) > 0
    assert hazards(asm) == []
