"""Frequencies stretched for long contexts against the formulas, pair by pair, over lengths from a few turns of the fastest pair to many of the slowest."""

import math

import pytest

from tilefish_b200 import TilefishPreconditionError
from tilefish_b200 import attention as A


def ramp_by_index(rot, base, length, factor, low, high):
    """Kept share of each pair's frequency: 1 up to the index that turns ``high`` times over ``length``, 0 from the one that turns ``low`` times on, a line between
    them over whole indexes. The line's end is an index of the formula, not of a pair: it may lie anywhere below ``rot``."""
    index = lambda turns: rot * math.log(length / (2 * math.pi * turns)) / (2 * math.log(base))  # noqa: E731
    begin, end = max(math.floor(index(high)), 0), min(math.ceil(index(low)), rot - 1)
    out = []
    for i in range(rot // 2):
        if i <= begin or i >= end:
            out.append(1.0 if i <= begin else 0.0)
        else:
            out.append((end - i) / (end - begin))
    return out


@pytest.mark.parametrize("rot,base", [(32, 10000.0), (64, 10000.0), (128, 10000.0), (128, 500000.0), (2, 10000.0), (6, 100.0)])
@pytest.mark.parametrize("length", [256, 4096, 54000, 65536, 131072, 262144, 10**7])
@pytest.mark.parametrize("low,high", [(1.0, 32.0), (0.25, 8.0)])
def test_yarn_is_the_formula_at_every_length(rot, base, length, low, high):
    factor = 4.0
    got, magnitude = A.rotary_frequencies(rot, base=base, scaling="yarn", factor=factor, length=length, low=low, high=high)
    assert magnitude == 0.1 * math.log(factor) + 1.0
    for i, keep in enumerate(ramp_by_index(rot, base, length, factor, low, high)):
        plain = base ** (-2.0 * i / rot)
        want = plain * keep + plain / factor * (1 - keep)
        assert abs(got[i] - want) <= 1e-13 * want, i


@pytest.mark.parametrize("length", [65536, 262144, 10**8])
def test_yarn_keeps_what_turns_often_to_the_last_pair(length):
    """A pair is divided by the whole factor only where it makes fewer than ``low`` turns."""
    rot, base = 64, 10000.0
    plain, _ = A.rotary_frequencies(rot, base=base)
    got, _ = A.rotary_frequencies(rot, base=base, scaling="yarn", factor=4.0, length=length)
    for f, g in zip(plain, got):
        turns = length * f / (2 * math.pi)
        assert (g > f / 4 * (1 + 1e-12)) == (turns > 1.0), (turns, g / f)
        if turns >= 32.0 * base ** (2 / rot):  # the line begins at a whole index, at most one below
            assert g == f


def test_yarn_divides_all_that_turn_less_than_low():
    """``length`` below one turn of the fastest pair: nothing is kept."""
    got, _ = A.rotary_frequencies(8, scaling="yarn", factor=2.0, length=6, low=1.0, high=32.0)
    assert got == [f / 2 for f in A.rotary_frequencies(8)[0]]


@pytest.mark.parametrize("base", [1.0, 0.5])
def test_yarn_refuses_a_base_without_a_slowest_pair(base):
    with pytest.raises(TilefishPreconditionError) as e:
        A.rotary_frequencies(64, base=base, scaling="yarn", factor=2.0, length=4096)
    assert e.value.kind == "argument" and e.value.arg == "base"
    assert len(A.rotary_frequencies(64, base=base)[0]) == 32
