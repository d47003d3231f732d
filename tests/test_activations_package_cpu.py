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


def test_two_outputs_in_one_place_are_refused():
    """da and db, the two outputs of a rotation or norm, and the two gains' gradients are written
    at once: in one place they would be a mixture."""
    import ctypes

    from ark_b200 import _lib
    L, by = _lib.lib(), ctypes.byref
    p = [0x7F0000000000 + (i << 24) for i in range(8)]      # aligned addresses that nothing reads
    plan = _lib.RopePlan()
    assert L.ark_cuda_rope_plan(by(plan), 64, 0, 10000.0, 0, 1.0, 0.0, 32.0, 1.0) == 0

    def heads(x):
        return by(_lib.Heads(x, 4, 256, 64))

    def rope(q, k, oq, ok, tokens=8, pos=p[6] + 4):         # a call that passes ends at the positions
        return L.ark_cuda_rope(by(plan), heads(q), heads(k), heads(oq), heads(ok), 0, tokens, 64, pos, 4, 0, 0, None)

    def back(oq, ok, gq, gk, ws=p[7] + 2):                  # or at the workspace
        return L.ark_cuda_qk_norm_rope_backward(
            by(plan), heads(p[0]), heads(p[1]), heads(oq), heads(ok), 0, 8, 64, None, None, heads(p[2]), heads(p[3]),
            p[4], p[4], 0, 1e-6, None, 0, 8, gq, gk, 0, 0, ws, L.ark_cuda_qk_norm_rope_workspace(64), None)

    assert back(p[0], p[1], p[4], p[5]) == -2 and back(p[0], p[1], p[4], p[4]) == -1
    assert back(p[6], p[6], p[4], p[5]) == -1 and back(p[1], p[0], p[4], p[5]) == -1
    assert back(p[1], p[6], p[4], p[5]) == -1
    for bad in ((p[0], p[1], p[2], p[2]), (p[0], p[1], p[1], p[2]), (p[0], p[1], p[2], p[0]), (p[0], p[0], p[0], p[2])):
        assert rope(*bad) == -1
    assert rope(p[0], p[1], p[0], p[1]) == rope(p[0], p[0], p[1], p[2]) == -2
    a = _lib.Act8(p[0], p[1], 8, 128, 0, 0)
    sw = lambda da, db: L.ark_cuda_swiglu_backward(p[2], 128, 0, by(a), by(a), da, 128, db, 128, None, None)  # noqa: E731
    assert sw(p[3], p[3]) == -1 and sw(p[3], p[4] + 1) == -2
    assert rope(p[0], p[1], p[2], p[2], tokens=0, pos=p[6]) == 0
