"""Angles of far positions, against thetas and turns in 50 digits.

Bounds: as for near positions (a float32 angle, cosine and sine, products and
sums: 6e-7 of |a| + |b|), and 2^-65 of a turn a position for theta's fixed
point."""
import decimal
import math

import pytest
import torch

from jasper_b200 import paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_far_positions(cuda, layout):
    r = paged.Rotary(32, layout=layout)
    positions = [2 ** 30 + 1, 2 ** 31 - 1, -2 ** 31, 10 ** 10 + 7, 2 ** 36 - 3, 2 ** 39, -2 ** 39 + 5, 2 ** 48 + 11]
    with decimal.localcontext() as c:
        c.prec = 50
        pi = decimal.Decimal("3.1415926535897932384626433832795028841971693993751058")
        turns = [[float(p * decimal.Decimal(10_000) ** (decimal.Decimal(-i) / 16) / (2 * pi) % 1) for i in range(16)]
                 for p in positions]
    angle = torch.tensor(turns, dtype=torch.float64)[:, None] * (2 * math.pi)
    x = torch.randn(len(positions), 5, 32, generator=torch.Generator().manual_seed(8))
    got = r.apply(x.cuda(), torch.tensor(positions, device="cuda")).cpu().double()
    x = x.double()
    first, second = (slice(0, 16), slice(16, 32)) if layout == "half" else (slice(0, 32, 2), slice(1, 32, 2))
    a, b = x[..., first], x[..., second]
    cos, sin = torch.cos(angle), torch.sin(angle)
    bound = (6e-7 + torch.tensor(positions).abs().double() * 2.0 ** -65 * 2 * math.pi)[:, None, None] * (a.abs() + b.abs())
    assert ((got[..., first] - (a * cos - b * sin)).abs() <= bound).all()
    assert ((got[..., second] - (b * cos + a * sin)).abs() <= bound).all()
