"""The angles of a rotation near the multiples of a quarter turn, against arithmetic of 60 digits: cosines and sines keep their relative accuracy."""

import math
from fractions import Fraction

import pytest
import torch

pytestmark = pytest.mark.gpu

TWO_PI = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")


@pytest.fixture(scope="module")
def A():
    from tilefish_b200 import attention, kernels

    kernels.require_cuda()
    return attention


def cos_sin(position, f):
    """In 64 bits, of the exact angle: what is left of the nearest quarter turn is small, and exact to 64 bits."""
    turn = position * Fraction(f) / TWO_PI
    turn -= math.floor(turn)
    quarter = round(4 * turn)
    rest = float((turn - Fraction(quarter, 4)) * TWO_PI)
    c, s = math.cos(rest), math.sin(rest)
    return [(c, s), (-s, c), (-c, -s), (s, -c)][quarter % 4]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("dim", [32, 34])  # whole vectors, and single pairs
def test_near_quarter_turns(A, layout, inverse, dim):
    inv = [math.pi / 2, math.pi, 2 * math.pi, 3 * math.pi / 2, math.pi / 4, 1.0, 0.1, 1e-3, 1e-6, 1e-9, math.pi / 2 + 1e-7, math.pi + 1e-6, math.pi / 2 - 3e-5, 0.7, 22.0, 355.0]
    positions = [0, 1, 2, 3, 4, 5, 7, 22, 355, 711, 4097, 65537, 131071, 10**6 + 3, 2**20 - 1, -1, -2, -3, -355, -70001]
    half = len(inv)
    i = torch.arange(half)
    i0, i1 = (i, i + half) if layout == "half" else (2 * i, 2 * i + 1)
    x = torch.zeros((len(positions), 2, dim))
    x[:, 0, i0], x[:, 1, i1] = 1.0, 1.0  # results are the cosines and sines themselves
    out = A.rotary(x.cuda(), torch.tensor(positions).cuda(), A.RotaryTable(inv, layout=layout), inverse=inverse).double().cpu()
    want = torch.tensor([[cos_sin(p, f) for f in inv] for p in positions], dtype=torch.float64)
    c, s = want[..., 0], want[..., 1] * (-1 if inverse else 1)
    # One step of an f32 for the function's value, half a step of what is left of the angle (that and the value differ by at most pi / 4 / sin(pi / 4) = 1.12), and
    # 2^-65 turns times the position for the table's frequency.
    bound = lambda t: t.abs() * (2.0**-23 + 1.12 * 2.0**-24) + 2.0**-62 * torch.tensor(positions).abs()[:, None]  # noqa: E731
    for got, exact in ((out[:, 0, i0], c), (out[:, 0, i1], s), (out[:, 1, i0], -s), (out[:, 1, i1], c)):
        assert ((got - exact).abs() <= bound(exact)).all(), ((got - exact).abs() / bound(exact)).max()
