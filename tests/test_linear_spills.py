"""What the assembler reports of linear attention's chunked kernels: registers spilled in them cost every call (at d = 64,
40 bytes of stores and 284 of loads made 8 x 8192 tokens, 32 heads, 422 us instead of 340)."""

import re
import subprocess

import pytest

from memt_b200 import build


@pytest.fixture(scope="module")
def spills(tmp_path_factory):
    try:
        nvcc = build._nvcc()
    except RuntimeError:
        pytest.skip("no nvcc")
    obj = tmp_path_factory.mktemp("linear") / "linear.o"
    r = subprocess.run([nvcc, *build.ARCH, *build.FLAGS, "-Xptxas", "-v", "-c", str(build.CSRC / "linear.cu"), "-o", str(obj)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    found = re.findall(r"Function properties for (\S+)\n\s+\d+ bytes stack frame, (\d+) bytes spill stores, (\d+) bytes",
                       r.stderr)
    return {name: (int(stores), int(loads)) for name, stores, loads in found}


# <D, whether outputs are made>: bytes of stores and loads that are left
@pytest.mark.parametrize("D,out,most", [(64, 1, (0, 0)), (64, 0, (0, 0)), (128, 1, (0, 0)), (128, 0, (4, 16)),
                                        (256, 1, (178, 168)), (256, 0, (0, 0))])
def test_chunked_kernels_spill_no_more(spills, D, out, most):
    of = [x for name, x in spills.items() if f"linear_tc_kernelILi{D}ELb{out}E" in name]
    assert len(of) == 1 and of[0][0] <= most[0] and of[0][1] <= most[1], of
