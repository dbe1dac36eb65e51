"""The tree and beam kernels keep their values in registers.

A value that the compiler spills inside a divergent branch can be stored under
that branch's lane mask and read back under the full one: in a form of the tree
kernel that spilled, the ring pointers of its path for values that are not finite
were garbage in the other lanes, and it read through them.  So no kernel of these
files may spill or use scratch memory."""
import os
import re
import subprocess

import pytest

from mockbird_amd import build


@pytest.mark.parametrize("source", ["tree.hip", "beam.hip"])
def test_no_kernel_spills(source, tmp_path):
    out = tmp_path / "k.s"
    subprocess.run([build.HIPCC, *build.HIP_FLAGS, "--cuda-device-only", "-S",
                    os.path.join(build.CSRC, source), "-o", str(out)], check=True,
                   capture_output=True)
    text = out.read_text()
    names = re.findall(r"^    \.name:\s+(\S+)", text, re.M)
    kernels = [n for n in names if n.startswith("_ZN2mb")]
    assert len(kernels) >= 6
    for field in (".private_segment_fixed_size", ".vgpr_spill_count"):
        values = re.findall(r"^    " + re.escape(field) + r":\s+(\d+)", text, re.M)
        assert len(values) == len(kernels)
        assert not any(map(int, values)), list(zip(kernels, values))
