"""rotate_heads on the GPU: what is said of second derivatives, the bounds of its angles, sines and cosines, and the way of large calls (several heads and several tiles of a CTA) against the definition."""
import warnings

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


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
