"""A rotation's table is what was checked when it was made."""

import copy

import pytest
import torch

from tilefish_b200 import attention as A


@pytest.mark.parametrize("name,value", [("rot", 64), ("turns", torch.zeros(1, dtype=torch.int64)), ("index", 0), ("layout", "interleaved"), ("magnitude", 1e300), ("_layout", 7)])
def test_nothing_of_a_table_is_exchanged(name, value):
    table = A.RotaryTable([1.0, 0.5], device="cpu")
    with pytest.raises(AttributeError, match=name):
        setattr(table, name, value)
    assert (table.rot, table.layout, table.magnitude, table.index, table._layout) == (4, "half", 1.0, -1, A.LAYOUTS["half"]) and table.turns.tolist() == A._turns([1.0, 0.5])


def test_a_subclass_has_attributes_of_its_own():
    class Named(A.RotaryTable):
        pass

    table = Named([1.0], device="cpu")
    table.name = "first"
    with pytest.raises(AttributeError, match="rot"):
        table.rot = 8
    other = copy.deepcopy(table)
    assert other.name == "first" and other.rot == 2


def test_copies():
    table = A.RotaryTable([1.0, 0.5], layout="interleaved", magnitude=1.5, device="cpu")
    for other in (copy.copy(table), copy.deepcopy(table)):
        assert (other.rot, other.layout, other.magnitude, other.index, other._layout) == (4, "interleaved", 1.5, -1, A.LAYOUTS["interleaved"]) and torch.equal(other.turns, table.turns)
