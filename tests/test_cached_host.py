"""CPU tests of h3q.cached's positions: places that come from device values stay inside the tables that they index."""
import pytest
import torch

import h3q
from h3q import cached


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


def test_positions():
    past = i32(5, 0, 9)
    assert cached.positions(past, 6).tolist() == [5, 6, 0, 1, 9, 10]
    assert cached.positions(past, 5, i32(0, 2, 2, 5)).tolist() == [5, 6, 9, 10, 11]
    assert cached.positions(past, 0).tolist() == []
    assert cached.positions(past[:0], 0, i32(0)).tolist() == []


def test_positions_of_tokens_of_no_sequence():
    """A padded step: starts ends before the tokens do, or begins behind the first."""
    past = i32(5, 0)
    assert cached.positions(past, 8, i32(0, 2, 5))[:5].tolist() == [5, 6, 0, 1, 2]
    got = cached.positions(past, 8, i32(3, 4, 8))
    assert got[3:].tolist() == [5, 0, 1, 2, 3] and got.numel() == 8


def test_tokens_without_a_sequence():
    for starts in (None, i32(0)):
        with pytest.raises(h3q.H3QError):
            cached.positions(i32(), 3, starts)


@pytest.mark.parametrize("past", [[0, 3], [7, 400], [-5, 2], [2**31 - 1, -(2**31)]])
@pytest.mark.parametrize("starts", [None, [0, 2, 4], [0, 1, 2], [1, 2, 3]])
def test_rope_rows_stay_inside_the_table(past, starts):
    rope = torch.arange(2 * 10 * 4, dtype=torch.float32).view(2, 10, 4)
    starts = None if starts is None else i32(*starts)
    pos = cached.positions(i32(*past), 4, starts)
    got = cached._rope_rows(rope, i32(*past), 4, starts)
    assert got.shape == (2, 4, 4) and got.is_contiguous()
    for i in range(4):
        assert torch.equal(got[:, i], rope[:, min(9, max(0, int(pos[i])))])


def test_rope_refusals():
    for rope in (torch.zeros(2, 0, 4), torch.zeros(10, 4), torch.zeros(1, 10, 4)):
        with pytest.raises(h3q.H3QError):
            cached._rope_rows(rope, i32(0), 1, None)
