"""CPU: no kernel's launch rule has a number of SMs in it; the device is asked (launch.cuh: sm_count)."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gemm4-attention-kernels_b200", "csrc")


def test_launch_rules_ask_the_device():
    found = []
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))):
        code = re.sub(r"//[^\n]*|/\*.*?\*/", "", open(path).read(), flags=re.S)
        found += [(os.path.basename(path), line.strip()) for line in code.splitlines() if re.search(r"\b148\b", line)]
    # what sm_count() returns where the device does not answer
    assert [f for f in found if not (f[0] == "launch.cuh" and "return 148;" in f[1])] == []
