"""CPU tests of rotate_heads: its oracle, the table of steps, and the entry points' checks of arguments."""
import ctypes
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

from oracle import rotate_oracle as ro


@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_gradients_equal_differences(interleaved):
    rng = np.random.default_rng(0)
    rot = ro.rotation(32, 16, sections=(3, 5), interleaved=interleaved)
    x, w, dy = rng.standard_normal((2, 3, 4, 32)), 1 + rng.standard_normal(32), rng.standard_normal((2, 3, 4, 32))
    pos = rng.integers(-50, 50, (2, 2, 4))
    dx, dw, _, _ = ro.backward(rot, x, dy, pos, w)
    f = lambda x, w: (ro.forward(rot, x, pos, w)[0] * dy).sum()  # noqa: E731
    for _ in range(20):
        i = tuple(rng.integers(0, n) for n in x.shape)
        step = np.zeros_like(x)
        step[i] = 1e-5
        # central differences of a smooth function: an error of some step^2, and of 2^-53 of the sum over the step
        assert abs((f(x + step, w) - f(x - step, w)) / 2e-5 - dx[i]) < 1e-6
        step = np.zeros_like(w)
        step[i[3]] = 1e-5
        assert abs((f(x, w + step) - f(x, w - step)) / 2e-5 - dw[i[3]]) < 1e-6


def test_oracle_is_a_rotation_that_depends_on_the_distance():
    rng = np.random.default_rng(1)
    rot = ro.rotation(16)
    q, k = rng.standard_normal((2, 1, 1, 1, 16))
    at = lambda p: np.array([[[p]]])  # noqa: E731
    scores = [float((ro.forward(rot, q, at(p + 7))[0] * ro.forward(rot, k, at(p))[0]).sum()) for p in (0, 5, 1000, 2 ** 30)]
    assert max(scores) - min(scores) < 1e-9
    assert np.allclose(np.linalg.norm(ro.forward(rot, q, at(12345))[0]), np.linalg.norm(q))


def test_steps_are_fractions_of_a_turn():
    from kerneldev_b200.rotate import _steps
    for f in (1.0, 0.5, 1e-3, 3.7, -1.0, 6.283185307179586, 0.0, 12345.678, 2.0 ** -60):
        step = _steps([f])[0]
        assert -2 ** 63 <= step < 2 ** 63
        turns = Fraction(step, 2 ** 64)
        for p in (1, 1000, 2 ** 31 - 1, -2 ** 31):
            angle = float(turns * p % 1) * 2 * math.pi
            want = float(np.fmod(np.longdouble(p) * np.longdouble(f), ro.TWO_PI))
            diff = abs(angle - want) % (2 * math.pi)
            # 2^-65 of a turn for each step, and the 64 bits of numpy's product where the angle is large
            assert min(diff, 2 * math.pi - diff) < 1e-9 + abs(p) * (2.0 ** -64 * 6.3 + abs(f) * 2.0 ** -63)
    with pytest.raises(ValueError, match="finite"):
        _steps([float("inf")])


def test_rotation_refuses_what_it_cannot_be():
    from kerneldev_b200 import Rotation
    for args, text in (({"head_dim": 24}, "head_dim"), ({"head_dim": 144}, "head_dim"), ({"head_dim": 64, "rotary_dim": 8}, "rotary_dim"), ({"head_dim": 64, "rotary_dim": 80}, "rotary_dim"),
                       ({"head_dim": 64, "sections": (16, 15)}, "sections"), ({"head_dim": 64, "sections": (8, 8, 8, 8)}, "sections"), ({"head_dim": 64, "sections": (-1, 33)}, "sections"),
                       ({"head_dim": 64, "sections": ()}, "sections"), ({"head_dim": 64, "base": 0.0}, "base"), ({"head_dim": 64, "frequencies": [1.0] * 31}, "frequencies"),
                       ({"head_dim": 16, "frequencies": [float("nan")] * 8}, "finite")):
        with pytest.raises(ValueError, match=text):
            Rotation(**args)
    with pytest.raises(RuntimeError, match="no CPU path"):
        Rotation(64, device="cpu")


def test_entry_points_reject_bad_arguments_before_touching_cuda():
    from kerneldev_b200 import _capi as m
    lib, p, n = m.load(), m.KdRotation(), ctypes.c_size_t(1)
    ref = ctypes.byref

    def refused(code, text, call=lib.kd_rotate):
        assert call(ref(p), None) == code and text in lib.kd_last_error(), lib.kd_last_error()

    assert lib.kd_rotate(None, None) == -1 and lib.kd_rotate_grad(None, None) == -1
    p.B, p.T, p.Hq, p.Hk, p.D, p.R, p.dtype, p.w_dtype, p.axes, p.eps, p.steps = 2, 3, 4, 1, 64, 64, m.KD_BF16, m.KD_F32, 1, 1e-6, 0x10000
    for name, value, code, text in (("B", -1, -1, b"shape"), ("Hq", 0, -1, b"shape"), ("Hk", -1, -1, b"shape"), ("T", -1, -1, b"shape"), ("D", 72, -1, b"head dim"), ("D", 144, -1, b"head dim"),
                                    ("R", 0, -1, b"rotated"), ("R", 80, -1, b"rotated"), ("R", 24, -1, b"rotated"), ("dtype", 5, -1, b"dtype"), ("w_dtype", -1, -1, b"dtype"), ("axes", 0, -1, b"axes"),
                                    ("axes", 4, -1, b"axes"), ("axes", 2, -1, b"positions"), ("positions", 0x10000, -1, b"no axis"), ("eps", -1.0, -1, b"eps"), ("eps", float("nan"), -1, b"eps"),
                                    ("steps", None, -1, b"steps"), ("steps", 0x10004, -2, b"steps"), ("T", 1 << 30, -4, b"tokens")):
        old = getattr(p, name)
        setattr(p, name, value)
        refused(code, text)
        refused(code, text, lib.kd_rotate_grad)
        setattr(p, name, old)
    refused(-1, b"q, its output")
    p.q.ptr = p.q_out.ptr = 0x10000
    refused(-1, b"k, its output")
    p.k.ptr, p.k_out.ptr = 0x10000, 0x10008
    refused(-2, b"16")
    p.k_out.ptr, p.q.stride_h = 0x10000, 3
    refused(-2, b"16")
    p.q.stride_h = 0
    p.dq.ptr = 0x10000
    refused(-1, b"k, its output", lib.kd_rotate_grad)
    p.dk.ptr, p.dq_weight = 0x10000, 0x10000
    refused(-1, b"not there", lib.kd_rotate_grad)
    p.q_weight = 0x10000
    refused(-1, b"workspace", lib.kd_rotate_grad)
    p.workspace = 0x10008
    refused(-2, b"workspace", lib.kd_rotate_grad)
    assert lib.kd_rotate_grad_workspace(ref(p), None) == -1
    assert lib.kd_rotate_grad_workspace(ref(p), ref(n)) == 0 and n.value >= 2 * 64 * 4
    p.T = 0
    assert lib.kd_rotate_grad_workspace(ref(p), ref(n)) == 0 and n.value == 0
    assert lib.kd_rotate(ref(p), None) == 0   # nothing to do
    refused(-1, b"no rows", lib.kd_rotate_grad)


def test_there_is_no_cpu_path():
    from kerneldev_b200 import rotate_heads
    from kerneldev_b200.rotate import _ext
    with pytest.raises(RuntimeError, match="no CPU path"):
        _ext.Rotation(torch.zeros(8, dtype=torch.int64), 16, False, [])
    with pytest.raises(ValueError, match="out_layout"):
        rotate_heads(torch.zeros(1, 1, 1, 16), None, None, out_layout="other")
