"""rotate_heads on the GPU: what is said of second derivatives, the bounds of its angles, sines and cosines, and the way of large calls (several heads and several tiles of a CTA) against the definition."""
import warnings

import numpy as np
import pytest
import torch

from oracle import rotate_oracle as ro
from tests.test_gpu_rotate import DT, HALF, assert_within, make, wide

pytestmark = pytest.mark.gpu
DEV = "cuda"


def turned_units(freq, positions):
    """Cosines and sines that the kernel forms for float32 heads: pairs (1, 0) turned, which multiplies with 1 and adds 0."""
    from kerneldev_b200 import Rotation, rotate_heads
    x = torch.zeros((1, 1, len(positions), 2 * len(freq)), device=DEV)
    x[..., :len(freq)] = 1
    y = wide(rotate_heads(x, None, Rotation(2 * len(freq), frequencies=list(freq), device=DEV), torch.tensor(positions, device=DEV)[None])[0])[0, 0]
    return y[:, :len(freq)], y[:, len(freq):]


def test_angles_are_rounded_to_the_nearest():
    """Angles of a few 2**-32 turns, whose sines show them: off by half of that, by 2**-65 turns for each step of the position, and by 2**-22 of themselves (the float nearest to 2 pi, a product, the sine's sum)."""
    rng = np.random.default_rng(0)
    freq, at = 2 * np.pi * 2.0 ** -32 * rng.uniform(-3, 3, 64), np.array([0, 1, -1, 2, 3, 5, -7, 11, 100, -255])
    _, s = turned_units(freq, at)
    want = np.sin(at[:, None] * freq)
    assert (np.abs(s - want) <= 2 * np.pi * (2.0 ** -33 + np.abs(at)[:, None] * 2.0 ** -65) + np.abs(want) * 2.0 ** -22).all()


def test_sines_and_cosines_of_float32_heads():
    """To 2**-23, as documented: in all quarters, at their borders and middles, near and far."""
    rng = np.random.default_rng(1)
    freq = np.concatenate((ro.rotation(48)["freq"], rng.uniform(-7, 7, 24), np.pi / 4 * np.array([1, -1, 2, -2, 3, 4, 1 + 2 ** -20, 1 - 2 ** -20, 2 + 2 ** -22, 0.5, 5, 7, -5, 6, 8, 0])))
    at = np.concatenate((np.arange(-1000, 1000), rng.integers(-2 ** 31, 2 ** 31, 2000), [2 ** 31 - 1, -2 ** 31]))
    angle = ro.angles({"freq": freq, "axis": np.zeros(64, int)}, at[None, None])[0]
    for got, want in zip(turned_units(freq, at), (np.cos(angle), np.sin(angle))):
        assert float(np.abs(got - want).max()) <= 2.0 ** -23


def test_second_derivatives_are_not_lost_without_a_word():
    """A warning where the gradients should have had a history, and an error where a loss with such gradients and other terms would lack their part."""
    from kerneldev_b200 import Rotation, rotate_heads
    rotation = Rotation(16, device=DEV)
    for which in ("", "q", "k", "qk"):
        q, k = (torch.randn((1, 2, 3, 16), device=DEV, requires_grad=True) for _ in range(2))
        weights = {f"{n}_weight": torch.ones(16, device=DEV, requires_grad=True) for n in which}
        a, b = rotate_heads(q, k, rotation, **weights)
        ordinary = a.square().sum() + b.square().sum()
        with pytest.warns(UserWarning, match="differentiable once"):
            g = torch.autograd.grad(ordinary, (q, k), create_graph=True)
        assert not any(x.requires_grad for x in g)
        with pytest.raises(RuntimeError, match="differentiable once"):
            (ordinary + sum(x.square().sum() for x in g)).backward()
        # the same call again, and twice where no second derivative is wanted
        a, b = rotate_heads(q, k, rotation, **weights)
        ordinary = a.square().sum() + b.square().sum()
        first = torch.autograd.grad(ordinary, (q, k), retain_graph=True)
        for x, y in zip(first, torch.autograd.grad(ordinary, (q, k))):
            assert torch.equal(x, y)


def test_no_word_where_nothing_is_lost():
    """Without norms, and with a gradient that depends on nothing, the rows' gradients do not either; nor do the weights' of rows that are not differentiated."""
    from kerneldev_b200 import Rotation, rotate_heads
    rotation = Rotation(16, device=DEV)
    x, dy = (torch.randn((1, 2, 3, 16), device=DEV) for _ in range(2))
    q, w = x.clone().requires_grad_(), torch.ones(16, device=DEV, requires_grad=True)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        y, _ = rotate_heads(q, None, rotation)
        for _ in range(2):
            torch.autograd.grad(y, q, dy, create_graph=True)
        y, _ = rotate_heads(x, None, rotation, q_weight=w)
        for _ in range(2):
            torch.autograd.grad(y, w, dy, create_graph=True)


# D, R, Hq, Hk, B, T, type, weights' type, layout, sections, interleaved, which weights
LARGE = [
    (64, 64, 4, 4, 3, 6007, "bf16", "bf16", "bthd", None, False, "qk"),
    (128, 64, 6, 3, 2, 6151, "f16", "f32", "bhtd", None, True, "qk"),
    (80, 80, 4, 2, 2, 8009, "f32", "f32", "bthd", (8, 16, 16), False, "qk"),
    (64, 64, 4, 4, 1, 16411, "f32", "f32", "bhtd", None, False, ""),
    (48, 32, 3, 3, 2, 12011, "bf16", "f32", "bthd", (5, 11), True, "k"),
    (128, 128, 8, 8, 1, 4099, "f32", "bf16", "bthd", None, False, "q"),
]


@pytest.mark.parametrize("case", LARGE, ids=lambda c: f"d{c[0]}r{c[1]}-{c[6]}-{c[2]}+{c[3]}")
def test_calls_of_several_heads_and_tiles_of_a_cta(case):
    """What large calls do: a thread has five rows and more, of several heads and several tiles of tokens, which go round its ring. Tolerances as in tests/test_gpu_rotate.py; chains of the weights' sums are
    at most 12 rows of a thread, 256 threads of a column, 10 CTAs of a lane and 32 lanes: 310 additions. Rows of float32 without a norm: the pair's length times 2**-22.5 for sine and cosine together, 2**-24 for
    the product that is rounded before the sum, 2**-30 for the angle: below 2**-22."""
    import ctypes

    from kerneldev_b200 import Rotation, _capi, rotate_heads
    D, R, Hq, Hk, B, T, dtype, wtype, layout, sections, interleaved, which = case
    p, n = _capi.KdRotation(), ctypes.c_size_t()
    p.B, p.T, p.Hq, p.Hk, p.D, p.R, p.dtype, p.w_dtype, p.axes, p.eps, p.steps = B, T, Hq, Hk, D, R, {"f16": _capi.KD_F16, "bf16": _capi.KD_BF16, "f32": 2}[dtype], 2, 1, 1e-6, 0x10000
    p.dq_weight = 0x10000
    assert _capi.load().kd_rotate_grad_workspace(ctypes.byref(p), ctypes.byref(n)) == 0
    ctas, rows = n.value // (4 * D), (Hq + Hk) * B * T // (8 * (32 // (D // 16)))   # rows: of all threads' groups, in tiles
    assert ctas <= 296 and rows >= 5 * ctas

    q, k, w, pos = make(case, seed=7)
    rotation, rot = Rotation(D, R, sections=sections, interleaved=interleaved, device=DEV), ro.rotation(D, R, sections=sections, interleaved=interleaved)
    leaves = [t.requires_grad_() for t in (q, k, w["q"], w["k"]) if t is not None]
    positions = torch.tensor(pos, device=DEV, dtype=torch.int32)
    out = rotate_heads(q, k, rotation, positions if sections else positions[0], q_weight=w["q"], k_weight=w["k"], out_layout="input")
    g = [torch.randn(y.shape, device=DEV).to(DT[dtype]) for y in out]
    got = dict(zip((id(t) for t in leaves), torch.autograd.grad(out, leaves, g)))
    for name, x, y, dy in zip("qk", (q, k), out, g):
        weight = None if w[name] is None else wide(w[name])
        exact = dtype == "f32" and weight is None
        want, size = ro.forward(rot, wide(x), pos, weight)
        assert_within(y, want, size * 2.0 ** (-22 if exact else -19) + np.abs(want) * HALF[dtype] + 1e-7 * (dtype == "f16"), name)
        dx, dw, big, sums = ro.backward(rot, wide(x), wide(dy), pos, weight)
        assert_within(got[id(x)], dx, big * 2.0 ** (-22 if exact else -18) + np.abs(dx) * HALF[dtype] + 1e-7 * (dtype == "f16"), "d" + name)
        if dw is not None:
            assert_within(got[id(w[name])], dw, sums * 2.0 ** -14 + np.abs(dw) * HALF[wtype] + 1e-7 * (wtype == "f16"), "d" + name + "_weight")
