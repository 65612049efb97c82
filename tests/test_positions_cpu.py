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


@pytest.mark.parametrize("shape", [(3, 5), (3, 5, 1), (15,)])
@pytest.mark.parametrize("dtype", [torch.bool, torch.float32, torch.uint8])
def test_positions_of_flags_in_any_shape(shape, dtype):
    """The scans take the flags of (B, T) steps in any shape of as many; so do the positions."""
    from memorax_b200.memoroid import episode_positions
    done = torch.tensor([[0, 0, 1, 0, 0], [1, 0, 0, 1, 1], [0, 0, 0, 0, 0]])
    start = torch.tensor([[7], [9], [2 ** 40]])
    want = torch.tensor([[7, 8, 0, 1, 2], [0, 1, 2, 0, 0], [2 ** 40 + i for i in range(5)]])
    assert torch.equal(episode_positions(done.to(dtype).reshape(shape), 3, 5, start, "cpu"), want)
    want[0, :2], want[2] = torch.tensor([0, 1]), torch.arange(5)
    assert torch.equal(episode_positions(done.to(dtype).reshape(shape), 3, 5, None, "cpu"), want)
