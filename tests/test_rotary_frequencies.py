"""Rotary frequencies to their last unit, against integer square roots."""
import decimal
import math

import pytest

from jasper_b200 import paged

BITS = 300


def inverse_roots(base, levels):
    """base ** (-1 / 2 ** j) for j = 0 .. levels, in units of 2^-BITS."""
    x = [(1 << BITS) // base]
    for _ in range(levels):
        x.append(math.isqrt(x[-1] << BITS))
    return x


def two_pi():
    """In units of 2^-BITS, from 16 atan(1/5) - 4 atan(1/239) (Machin)."""
    def atan(n):
        total, term, k = 0, (1 << (BITS + 20)) // n, 0
        while term:
            total += (-1) ** k * term // (2 * k + 1)
            term, k = term // (n * n), k + 1
        return total
    return (2 * (16 * atan(5) - 4 * atan(239))) >> 20


@pytest.mark.parametrize("base", [10_000, 500_000, 7])
@pytest.mark.parametrize("rot", [2, 4, 16, 64])
@pytest.mark.parametrize("factor", [1, 4])
def test_frequencies_are_rounded_once(base, rot, factor):
    kw = {} if factor == 1 else dict(scaling="linear", factor=factor)
    r = paged.Rotary(128, rot, base=base, device="cpu", **kw)
    levels = int(math.log2(rot)) - 1
    roots, circle = inverse_roots(base, levels), two_pi()
    for i, f in enumerate(r._freq.tolist()):
        theta = 1 << BITS                                   # base ** (-2 i / rot): i's bits pick the roots
        for j in range(levels + 1):
            if i >> (levels - j) & 1:
                theta = theta * roots[j] >> BITS
        exact = theta * 2 ** 64 * 2 ** 64 // (circle * factor)     # in units of 2^-64 of the last unit
        assert abs(f * 2 ** 64 - exact) <= 2 ** 63 + 2 ** 20
        assert abs(r.theta[i] - theta / 2 ** BITS / factor) <= 2.0 ** -53 * r.theta[i]


def test_scaled_frequencies_are_rounded_once():
    """ntk and yarn by their formulas in other precision."""
    with decimal.localcontext() as c:
        c.prec = 80
        pi = decimal.Decimal(two_pi()) / 2 / 2 ** BITS
        plain = [decimal.Decimal(10_000) ** (decimal.Decimal(-i) / 32) for i in range(32)]
        base = 10_000 * decimal.Decimal(8) ** (decimal.Decimal(64) / 62)
        low = math.floor(64 * math.log(4096 / (32 * 2 * math.pi)) / (2 * math.log(10_000)))
        high = math.ceil(64 * math.log(4096 / (2 * math.pi)) / (2 * math.log(10_000)))
        slow = [min(1, max(0, decimal.Decimal(i - low) / (high - low))) for i in range(32)]
        for want, kw in (([base ** (decimal.Decimal(-i) / 32) for i in range(32)], dict(scaling="ntk")),
                         ([t * (1 - s) + t / 8 * s for t, s in zip(plain, slow)],
                          dict(scaling="yarn", trained_length=4096))):
            got = paged.Rotary(64, factor=8.0, device="cpu", **kw)._freq.tolist()
            for f, t in zip(got, want):
                assert abs(f - t / (2 * pi) * 2 ** 64) <= decimal.Decimal("0.5000001")
