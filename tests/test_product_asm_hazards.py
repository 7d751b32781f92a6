"""The kernels of csrc/product.hpp issue their matrix instructions from assembly as the GEMM's do, and with the same two hazards, for which the
compiler does not know to wait: tests/test_gemm_asm_hazards.py says which.  Here their assembly is checked, and that nothing is spilled where
the matrix instructions are."""

import os
import re
import shutil
import subprocess
import tempfile

import pytest

from tests.test_gemm_asm_hazards import HIPCC, ROOT, _check

# kernels of csrc/<file>.hip: ring, columns, and both products of a gradient, by operand type and what becomes of the product
FILES = {"gemm_int8": (27, 0, 0), "gated_ffn": (14, 32, 8), "linear_cross_entropy": (36, 32, 8)}


@pytest.mark.skipif(not shutil.which(HIPCC), reason="hipcc not available")
def test_kernels_have_no_unprotected_mfma_hazards():
    with tempfile.TemporaryDirectory() as d:
        runs = {
            name: subprocess.Popen(
                [HIPCC, "-O3", "-std=c++20", "--offload-arch=gfx950", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", f"-I{ROOT}/include",
                 f"-I{ROOT}/tilefusion_amd/include", f"-I{ROOT}/tilefusion_amd/csrc", "-Wno-unused-command-line-argument", "--cuda-device-only", "-S",
                 "-x", "hip", f"{ROOT}/tilefusion_amd/csrc/{name}.hip", "-o", os.path.join(d, name + ".s")], stderr=subprocess.DEVNULL)
            for name in FILES}
        for name, kinds in FILES.items():
            assert runs[name].wait() == 0
            text = open(os.path.join(d, name + ".s")).read()
            kernels = re.findall(r"^(_ZN3tfk\S*product_(?:ring64|cols|pair)_kernel\S*):[^\n]*\n(.*?)\.section", text, flags=re.S | re.M)
            found = tuple(sum(f"product_{kind}_kernel" in k for k, _ in kernels) for kind in ("ring64", "cols", "pair"))
            assert found == kinds, f"{name}: {found}"
            for kernel, body in kernels:
                assert _check(kernel, body) >= 32, kernel
                lines = [line.strip() for line in body.splitlines() if line.strip() and not line.strip().startswith(";")]
                mfma = [i for i, line in enumerate(lines) if line.startswith("v_mfma")]
                loops = 2 if "product_pair_kernel" in kernel else 1   # (each has as many, and lies in one piece)
                for i in range(loops):
                    loop = mfma[i * len(mfma) // loops:(i + 1) * len(mfma) // loops]
                    assert not any(line.startswith("scratch_") for line in lines[loop[0]:loop[-1]]), f"{kernel}: spilled in the main loop"
