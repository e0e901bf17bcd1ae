"""No register of a layer operator's kernel lies in memory (CPU check: hipcc cross-compiles gfx950 and reports every kernel's resources). The attention kernels
count their transfers to LDS by hand, the 4-bit ones keep two rounds of loads in flight: a spilled register is a wait for all of them."""
import os
import re
import subprocess

import pytest

from shodh_memory_amd import build

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "shodh_memory_amd", "csrc")


@pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="no hipcc")
@pytest.mark.parametrize("source", ["rms_norm.hip", "dense_w4.hip", "window_attention.hip"])
def test_no_spills(source):
    out = subprocess.run([build.HIPCC] + build.FLAGS + ["-Rpass-analysis=kernel-resource-usage", "--cuda-device-only", "-c", os.path.join(CSRC, source), "-o", "/dev/null"],
                         capture_output=True, text=True, timeout=900)
    assert out.returncode == 0, out.stderr[-2000:]
    names = re.findall(r"Function Name: (\S+)", out.stderr)
    spills = [int(n) for n in re.findall(r"VGPRs Spill: (\d+)", out.stderr)]
    kernels = {n: s for n, s in zip(names, spills)}
    assert len(names) == len(spills) > 3
    assert not {n: s for n, s in kernels.items() if s}
