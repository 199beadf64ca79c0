"""CPU test of the rounding of 16-bit numbers to 4 bits, up to the largest quotient."""
import numpy as np


def test_product_with_a_rounded_inverse_decides_as_the_quotient_does_up_to_the_largest():
    """x times a float within 2**-22 of 1 / scale, on the grid of 2**-13 that a fused sum with 1536 leaves, is on the side of each middle of two levels that x / scale is on: for every x of 11 bits, every scale of
    4 bits and both their exponents (powers of two apart), with quotients beyond the last middle. (An x of 2047 / 32 ends below five for scales of 13, 14 and 15 eighths.)"""
    middles = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)
    x = np.arange(1024, 2048, dtype=np.float64)
    for m in range(8, 16):
        v = np.concatenate([x * 2.0 ** e for e in range(-30, -2)])
        v = v[v <= 6.5 * m]
        assert v.max() / m > 6.4 and all((v == middle * m).any() and ((v > middle * m) & (v < 1.01 * middle * m)).any() for middle in middles)
        nearest = np.float32(1) / np.float32(m)
        for inverse in (nearest, np.nextafter(nearest, np.float32(0)), np.nextafter(nearest, np.float32(1))):
            q = (v * np.float64(inverse) + 1536.0).astype(np.float32) - np.float32(1536)
            for middle in middles:
                assert np.array_equal(np.sign(q.astype(np.float64) - middle), np.sign(v - middle * m))
