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


def test_forward_mode_derivatives_are_refused():
    """The launch knows nothing of tangents: dropping one would be a derivative of zero."""
    import torch
    import torch.autograd.forward_ad as fwd

    from gear_b200 import _native as N
    from gear_b200 import core, recurrence
    x, g, h0 = torch.ones(2, 3, 4), torch.ones(2, 3, 4), torch.ones(2, 4)
    for at in range(3):
        with fwd.dual_level():
            t = [x, g, h0]
            t[at] = fwd.make_dual(t[at], torch.ones_like(t[at]))
            with pytest.raises(core.GearError, match="forward-mode") as e:
                recurrence.linear_recurrence(t[0], t[1], h0=t[2])
            assert e.value.code == N.ERR_INVALID
    for leaf in (x, g, h0):       # beside reverse mode, too
        leaf.requires_grad_(True)
    with fwd.dual_level(), pytest.raises(core.GearError, match="forward-mode"):
        recurrence.linear_recurrence(fwd.make_dual(x, torch.ones_like(x)), g, h0=h0)
    with fwd.dual_level(), pytest.raises(core.GearError, match="CUDA"):      # a level alone changes nothing
        recurrence.linear_recurrence(x, g, h0=h0)
    with pytest.raises(core.GearError, match="forward-mode"):
        torch.func.jvp(lambda t: recurrence.linear_recurrence(t, g.detach())[0], (x.detach(),), (x.detach(),))


@pytest.mark.parametrize("backward", [False, True])
def test_scratch_that_is_not_aligned_is_refused(backward):
    import ctypes as C

    from gear_b200 import _native as N
    a = N.RecurrenceArgs(x=256, gate=256, x_dtype=N.DT_F32, gate_dtype=N.DT_F32, batch=1, time=100, width=64, gates=64,
                         sequences=1, out=256, dout=256, dx=256, dgate=256, carry=256)
    scratch, carry = C.c_int64(0), C.c_int64(0)
    assert N.lib.gearb_recurrence_bytes(C.byref(a), int(backward), C.byref(scratch), C.byref(carry)) == N.OK
    a.scratch_bytes = scratch.value
    run = N.lib.gearb_recurrence_backward if backward else N.lib.gearb_recurrence_forward
    for at in (1, 4, 8, 15):
        a.scratch = 4096 + at
        assert run(C.byref(a), None) == N.ERR_INVALID
        assert "16 bytes" in N.lib.gearb_last_error().decode()


def test_layout_scratch_that_is_not_aligned_is_refused():
    import ctypes as C

    from gear_b200 import _native as N
    a = N.LayoutArgs(lengths=256, requests=3, page=16, max_blocks=4, block_table=256, num_pages=5, used_in=256, used_out=256,
                     offsets=256, scratch_bytes=N.lib.gearb_layout_scratch_bytes(3))
    for at in (1, 4):
        a.scratch = 4096 + at
        assert N.lib.gearb_layout_paged(C.byref(a), None) == N.ERR_INVALID
        assert "8 bytes" in N.lib.gearb_last_error().decode()
