"""Multi-axis rotation at far positions against angles in 60 decimal digits: the bound that the comments state."""
from decimal import Decimal, getcontext

import pytest
import torch

from pie_b200 import ops

PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
THETA, HALF = 500000, 64
POSITIONS = [0, 1, 250000, 2 ** 22, 2 ** 22 + 1, 2 ** 26 + 3, 2 ** 30, 2 ** 30 + 12345, 2 ** 31 - 2, 2 ** 31 - 1, -(2 ** 31), -(2 ** 30) - 7]


def _turns_per_position():
    """f_i / 2 pi of every pair, exact to 50 digits."""
    getcontext().prec = 60
    return [Decimal(THETA) ** (Decimal(-2 * i) / Decimal(2 * HALF)) / (2 * PI) for i in range(HALF)]


def _config():
    return ops.AxisRopeConfig(mode="plain", theta=float(THETA), scale=1.0, sections=(16, 24, 24))


def test_the_table_is_within_its_bound():
    table = _config().prepared()
    for i, want in enumerate(_turns_per_position()):
        got = Decimal(table.turn[i]) / Decimal(2 ** 64)
        # a power, the 2 pi it is divided by and the quotient round to 53 bits, the power by up to twice as much; the
        # fixed point drops what is below 2^-64
        assert abs(got - want) <= want * Decimal(2) ** -51 + Decimal(2) ** -64, i


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [len(POSITIONS), 200 * len(POSITIONS)])  # the kernel for few tokens and the one for many
def test_far_positions(tokens):
    turns = _turns_per_position()
    g = torch.Generator().manual_seed(3)
    x = torch.randn((tokens, 2, 128), generator=g)
    pos = torch.tensor(POSITIONS * (tokens // len(POSITIONS)), dtype=torch.int32)
    q, k = x.cuda(), x[:, :1].contiguous().cuda()
    ops.apply_rope_axes_inplace(q, k, pos.repeat(3, 1).cuda(), _config())
    cos, sin, angle = (torch.empty((len(POSITIONS), HALF), dtype=torch.float64) for _ in range(3))
    for a, p in enumerate(POSITIONS):
        for i, t in enumerate(turns):
            turn = p * t
            rest = float((turn - turn.to_integral_value()) * 2 * PI)  # within half a turn: 2^-53 of it is lost
            cos[a, i], sin[a, i] = torch.tensor(rest, dtype=torch.float64).cos(), torch.tensor(rest, dtype=torch.float64).sin()
            # what the angle may be off by, in turns: the frequency; 32 bits of a turn are kept, then 24 bits of up to 1/8
            angle[a, i] = abs(p) * float(t) * 2.0 ** -51 + abs(p) * 2.0 ** -64 + 2.0 ** -32 + 2.0 ** -28
    rows = torch.arange(tokens) % len(POSITIONS)
    c, s, off = cos[rows][:, None], sin[rows][:, None], 2 * 3.1416 * angle[rows][:, None]
    for got, src in ((q, x), (k, x[:, :1])):
        a, b = src[..., :HALF].double(), src[..., HALF:].double()
        want = torch.cat([a * c - b * s, a * s + b * c], -1)
        # cos and sin within 2^-23, two products and a sum of 2^-24 each, of |a| + |b|
        bound = ((a.abs() + b.abs()) * (off + 2.0 ** -23 + 2 * 2.0 ** -24)).repeat(1, 1, 2)
        worst = ((got.cpu().double() - want).abs() - bound).max().item()
        assert worst <= 0, worst
    assert ops.device_error("cuda") is None
