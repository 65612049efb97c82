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


@pytest.mark.parametrize("dim,base", [(64, 10000.0), (128, 500000.0), (8, 100.0)])
def test_a_position_below_2_to_40_keeps_its_angle(dim, base):
    """The phase of a position (the product with the plan's rate, modulo a turn) against 60 digits: off by at most half of 2^-64 of a turn
    for each step of the position."""
    import decimal
    from memorax_b200 import ops
    turns = ops.RotaryPlan(dim, base=base, device="cpu").turns.tolist()
    with decimal.localcontext() as ctx:
        ctx.prec = 60
        two_pi = decimal.Decimal("6.28318530717958647692528676655900576839433879875021164194988918461563281257")
        for i, t in enumerate(turns):
            rate = (-2 * i * decimal.Decimal(base).ln() / dim).exp() / two_pi
            for position in (1, 1000003, 2 ** 34 - 1, 2 ** 40 - 1, -(2 ** 40) + 5):
                off = abs(decimal.Decimal(position * t % 2 ** 64) / 2 ** 64 - rate * position) % 1
                assert min(off, 1 - off) <= decimal.Decimal(abs(position)) / 2 ** 65 * decimal.Decimal("1.001")
