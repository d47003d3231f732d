"""The activation operators beside the rest of the package: what was there
before their first use is there after it."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT


def run(code):
    return subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)


def test_lib_stays_a_function():
    r = run("import ark_b200 as ab\n"
            "before = ab.lib\n"
            "ab.Act8, ab.RopePlan, ab.weight_grad\n"
            "assert ab.lib is before and ab.lib().ark_cuda_act8_pitch(1) == 128\n"
            "from ark_b200 import lib\n"
            "assert lib is before\n")
    assert r.returncode == 0, r.stderr


def test_the_c_library_builds_without_torch():
    """`make` in a Python that has no torch: the commands for the library, none for the binding."""
    r = subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, "ark_b200", "csrc"),
                        f"PYTHON={sys.executable} -I -S"], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stderr == ""
    assert "libark_cuda.a" in r.stdout and "libark_cuda.so" in r.stdout
    assert "_ark_torch" not in r.stdout and "torch/include" not in r.stdout


def test_no_view_of_a_closed_optimizers_buffer():
    """close() gives the gradient buffer back: a range of it would be freed memory."""
    import torch

    import ark_b200 as ab
    from ark_b200 import layout
    opt = object.__new__(ab.Optimizer)
    opt.layout, opt._h = layout.decoder_layout("tiny", 1, 8, 16, 32), None
    opt._gbuf = torch.zeros(opt.layout.n)
    assert opt.grad_view("l0.w1").numel() == 128
    opt.close()
    with pytest.raises(RuntimeError, match="grad_buffer"):
        opt.grad_view("l0.w1")


def test_wide_checkpoints_need_room_for_both_halves():
    """FP16 dY with a checkpoint of a wider type: the workspace holds dY twice, and the call says
    so when it does not; a BF16 dY needs none of it."""
    import ctypes

    from ark_b200 import _lib
    L, p = _lib.lib(), 0x7F0000001000      # an aligned address that nothing reads
    narrow, wide = (_lib.Act8(p, p, 64, 100, 0, w) for w in (0, 1))
    need = [L.ark_cuda_weight_grad_workspace(ctypes.byref(x), p, 64, 64) for x in (narrow, wide)]
    assert need[1] >= need[0] + 2 * 64 * 64 * 2 + 100 * 64 * 4

    def call(x, ws, nbytes, dy_type=0):
        return L.ark_cuda_weight_grad(ctypes.byref(x), p, dy_type, 64, 64, p, 0, 64, 0, ws, nbytes, None)

    assert call(wide, None, 0) == -1 and call(wide, p, need[1] - 1) == -1
    assert call(wide, p + 8, need[1]) == -2
    if need[0]:
        assert call(wide, p, need[0] - 1, dy_type=1) == -1
