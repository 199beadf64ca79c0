"""rotate_heads on the GPU: what is said of second derivatives, the bounds of its angles, sines and cosines, and the way of large calls (several heads and several tiles of a CTA) against the definition."""
import warnings

import numpy as np
import pytest
import torch

from oracle import rotate_oracle as ro
from tests.test_gpu_rotate import wide

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
