"""Carries of the delta-rule cell with and without positions."""
import pytest
import torch


@pytest.fixture(scope="module")
def cells():
    from memorax_b200.build import build_library
    build_library()
    from memorax_b200.memoroid import DeltaNetCell
    return {"without": DeltaNetCell(8, 64, 1), "with": DeltaNetCell(8, 64, 1, rotary_base=10000.0)}


@pytest.mark.parametrize("of,given", [("without", "with"), ("with", "without")])
def test_a_carry_of_the_other_kind_is_refused(cells, of, given):
    """A position that a cell has no use for is not dropped, and one that it lacks is not made up."""
    cell, x, done = cells[of], torch.zeros(2, 3, 8), torch.zeros(2, 3)
    carry = cells[given].initialize_carry(None, (2, 8))
    for call in (lambda: cell.layer(x, done, carry), lambda: cell.bfloat16().layer(x.bfloat16(), done, carry), lambda: cell.scan((None,) * 4, carry, done, x)):
        with pytest.raises(ValueError, match="positions"):
            call()
    with pytest.raises(ValueError, match="positions"):
        cell.layer(x, done, ())
