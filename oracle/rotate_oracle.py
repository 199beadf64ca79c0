"""Norms of heads and their rotation by positions in 64 bits on the CPU (numpy), from the definition: what the GPU tests compare with.

A rotation is a dict: freq float64 (R / 2,), axis int (R / 2,), interleaved bool. Positions are int64 (axes, B, T).
"""
import numpy as np

TWO_PI = np.longdouble("6.283185307179586476925286766559005768394338798750211641949889")


def rotation(D, R=None, base=10000.0, freq=None, sections=None, interleaved=False):
    R = D if R is None else R
    if freq is None:
        freq = [base ** (-2.0 * i / R) for i in range(R // 2)]
    axis = [a for a, n in enumerate(sections or (R // 2,)) for _ in range(n)]
    return {"freq": np.asarray(freq, np.float64), "axis": np.asarray(axis, int), "interleaved": interleaved}


def angles(rot, positions):
    """(B, T, R / 2): the product in 64 bits of mantissa and without its whole turns: a far position's angle is as exact as a near one's."""
    p = np.asarray(positions)[rot["axis"]].transpose(1, 2, 0).astype(np.longdouble)
    return np.fmod(p * rot["freq"].astype(np.longdouble), TWO_PI).astype(np.float64)


def _pairs(rot):
    n = len(rot["freq"])
    i = np.arange(n)
    return (2 * i, 2 * i + 1) if rot["interleaved"] else (i, i + n)


def turn(rot, x, angle):
    """x (B, H, T, D) turned by angle (B, T, R / 2)."""
    a, b = _pairs(rot)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    y = x.copy()
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def size(rot, x):
    """What an element's error is relative to: the length of its pair."""
    a, b = _pairs(rot)
    y = np.abs(x)
    y[..., a] = y[..., b] = np.hypot(x[..., a], x[..., b])
    return y


def forward(rot, x, positions, weight=None, eps=1e-6):
    """(y, the lengths that its errors are relative to)."""
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight
    return turn(rot, x, angles(rot, positions)), size(rot, x)


def backward(rot, x, dy, positions, weight=None, eps=1e-6):
    """(dx, dw or None, and for both what their errors are relative to)."""
    g, most = turn(rot, dy, -angles(rot, positions)), size(rot, dy)
    if weight is None:
        return g, None, most, None
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    unit = x * r
    h = g * weight
    dx = r * (h - unit * (h * unit).mean(-1, keepdims=True))
    big = r * (most * np.abs(weight) + np.abs(unit) * (most * np.abs(weight * unit)).mean(-1, keepdims=True))
    return dx, (g * unit).sum((0, 1, 2)), big, (most * np.abs(unit)).sum((0, 1, 2))
