"""Host-side parts of the recurrences."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


def test_waits_that_leave_turns_out_end_behind_their_own_phase(tmp_path):
    """The ring rule of the streaming kernels' finishers, in every state their barriers may be in."""
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("g++ is needed")
    exe = tmp_path / "ring_model"
    build = subprocess.run([gxx, "-std=c++17", "-O1", "-I", str(ROOT / "gear_b200" / "csrc"),
                            str(ROOT / "tests" / "host" / "ring_model.cc"), "-o", str(exe)], capture_output=True, text=True)
    assert build.returncode == 0, build.stderr[-2000:]
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and "states ok" in run.stdout, run.stdout
