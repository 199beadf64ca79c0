"""Rotation of queries and keys by their positions, with the norms of their heads, ahead of the attention.

``GPTModel`` adds learned positions to its embeddings (model.py:152, :188-191), which end where they were trained. ``rotate_heads`` gives the queries and keys of
``flash_attention`` or of the cache relative positions instead: pairs of a head's elements turn by angles that grow with the position. In the
same pass it can divide each head's row by its root mean square and weight it, which keeps scores bounded. Both directions are one kernel each (and one for the
weights' gradients).

``rotate_heads`` stands between the projections and ``flash_attention`` or ``cache_append`` and ``cache_attention``::

    rotation = Rotation(head_dim, base=1e6)                                       # once
    q, k = rotate_heads(q, k, rotation, q_weight=wq, k_weight=wk)                 # training: positions 0 .. time - 1
    q, k = rotate_heads(q, k, rotation, offsets=lens, q_weight=wq, k_weight=wk)   # generating: behind the lens[b] tokens that a cache holds
"""
from __future__ import annotations

import math
from fractions import Fraction

import torch

from . import _host

_ext = _host.load()

__all__ = ["Rotation", "rotate_heads"]

# 1 / (2 pi) in 160 bits, from pi's first 60 decimals
_PI = Fraction("3.141592653589793238462643383279502884197169399375105820974944")
_TURN = int(Fraction(2) ** 160 / (2 * _PI))


def _steps(frequencies) -> list[int]:
    """Angles (radians for a step of the position) as fractions of 2**64 turns, nearest, as signed words."""
    out = []
    for f in frequencies:
        f = float(f)
        if not math.isfinite(f):
            raise ValueError("frequencies must be finite")
        a, b = f.as_integer_ratio()
        n = (2 * a * _TURN + (b << 96)) // (b << 97) % 2 ** 64   # whole turns make no difference
        out.append(n - 2 ** 64 if n >= 2 ** 63 else n)
    return out


class Rotation:
    """Which elements of a head turn, by what, and how far: made once, for any number of calls.

    head_dim: a multiple of 16 from 16 to 128. rotary_dim: the first so many elements turn, a multiple of 16; None: all. Pair i of them is elements
    i and i + rotary_dim / 2, or 2 i and 2 i + 1 with ``interleaved``, and turns by position * frequencies[i] radians; frequencies: rotary_dim / 2 numbers
    (scaled ones of a longer context, or those of several axes), by default base ** (-2 i / rotary_dim). sections: how many pairs turn by the first, second and third axis of the
    positions (time, height and width of a video's patches), rotary_dim / 2 together; None: there is one axis.

    Angles are exact to 2**-32 of a turn at any 32-bit position; sines and cosines to 2**-23 for float32 heads, 2**-20 for those of 16 bits."""

    __slots__ = ("head_dim", "rotary_dim", "interleaved", "sections", "steps", "_core")

    def __init__(self, head_dim: int, rotary_dim: int | None = None, base: float = 10000.0, frequencies=None, sections=None, interleaved: bool = False, device="cuda"):
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if head_dim % 16 or not 16 <= head_dim <= 128:
            raise ValueError(f"head_dim {head_dim} is not supported (a multiple of 16 from 16 to 128)")
        if rotary_dim % 16 or not 16 <= rotary_dim <= head_dim:
            raise ValueError(f"rotary_dim {rotary_dim} is not supported (a multiple of 16 from 16 to head_dim)")
        pairs = rotary_dim // 2
        sections = None if sections is None else tuple(int(n) for n in sections)
        if sections is not None and (not 1 <= len(sections) <= 3 or min(sections) < 0 or sum(sections) != pairs):
            raise ValueError(f"sections must be one to three counts of pairs, {pairs} together, got {sections}")
        if frequencies is None:
            if not (math.isfinite(base) and base > 0):
                raise ValueError("base must be positive and finite")
            frequencies = [base ** (-2.0 * i / rotary_dim) for i in range(pairs)]
        elif isinstance(frequencies, torch.Tensor):
            frequencies = frequencies.detach().double().cpu().flatten().tolist()
        if len(frequencies) != pairs:
            raise ValueError(f"frequencies must be {pairs} numbers, got {len(frequencies)}")
        steps = torch.tensor(_steps(frequencies), dtype=torch.int64)
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("rotate_heads runs on CUDA sm_100 devices only; there is no CPU path")
        self.head_dim, self.rotary_dim, self.interleaved, self.sections = head_dim, rotary_dim, bool(interleaved), sections
        self.steps = steps.to(device)
        self._core = _ext.Rotation(self.steps, head_dim, self.interleaved, list(sections or ()))


def rotate_heads(q: torch.Tensor, k: torch.Tensor | None, rotation: Rotation, positions: torch.Tensor | None = None, offsets: torch.Tensor | None = None,
                 q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6, out_layout: str = "contiguous"):
    """(q, k), each row normalised where its weight is given, and turned by its token's position.

    q (batch, heads, time, head_dim), k (batch, key heads, time, head_dim) or None: float16, bfloat16 or float32, any strides. positions: int32 or int64
    (batch, time), or (axes, batch, time) for a rotation with sections; a batch of 1 serves all sequences. offsets: int32 (batch,), the positions of a
    sequence's tokens are offsets[b], offsets[b] + 1, ... Neither: 0, 1, ... Both stay on the device, so that a step can be captured.

    q_weight, k_weight: (head_dim,) in any of the three types. With one, a row x becomes weight * x / sqrt(mean(x**2) + eps) before it is turned; the mean is taken in 32 bits
    (squares beyond its range make the row zeros; with an eps of 0 a row whose squares are all below it, or zero, becomes infinities and NaN). Everything is computed in 32 bits and rounded once.

    Differentiable, once, in q, k and the weights; sums over rows are taken in a fixed order. With ``create_graph`` the gradients are plain tensors all the same: where a second derivative would go through
    them a warning says so, and a later backward pass through the same call, as that of a loss with these gradients and other terms, is refused. A backward pass that adds to leaves cannot be captured while an
    earlier graph of the same leaves lives (it is refused). out_layout: "contiguous", or "input" for the outputs and gradients in the memory layouts of q and k."""
    if out_layout not in ("contiguous", "input"):
        raise ValueError("out_layout must be 'contiguous' or 'input'")
    return _ext.rotate_heads(q, k, rotation._core, positions, offsets, q_weight, k_weight, eps, out_layout == "input")
