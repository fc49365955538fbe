"""Kernels that stage copies in rings wait, before they give up, for the copies that are still under way: which phase of
each buffer's barrier that is, on the CPU; and that the kernels ask for that phase, not for either."""
import re
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent
KERNELS = ROOT / "ascend_mlir_b200" / "csrc" / "kernels"


def test_newest_fill(tmp_path):
    exe = tmp_path / "ring_drain"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-I", str(ROOT / "ascend_mlir_b200" / "csrc"),
                    str(ROOT / "tests" / "cpp" / "ring_drain.cpp"), "-o", str(exe)], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout


def test_no_wait_for_either_phase():
    """A condition that tries a barrier's two parities is over at once."""
    either = re.compile(r"mbarTryWait\(([^;{}]*?), 0\)\s*&&\s*!mbarTryWait\(([^;{}]*?), 1\)")
    found = {p.name for p in sorted(KERNELS.glob("*.cu*")) if either.search(p.read_text())}
    assert not found, found
