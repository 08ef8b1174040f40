"""Every kernel source is compiled without packed fp32 instructions (no GPU needed: make prints its commands)."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "dig_amd", "csrc")


def test_no_packed_fp32():
    out = subprocess.run(["make", "-n", "-B", "-C", CSRC], capture_output=True, text=True, check=True).stdout
    lines = [ln.split() for ln in out.splitlines() if " -c " in ln and ".hip " in ln]
    built = {w for ln in lines for w in ln if w.endswith(".hip")}
    assert built == {f for f in os.listdir(CSRC) if f.endswith(".hip")}
    for ln in lines:
        at = ln.index("-packed-fp32-ops")
        assert ln[at - 3:at] == ["-Xclang", "-target-feature", "-Xclang"], ln
