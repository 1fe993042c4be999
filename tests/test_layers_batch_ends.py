"""Which steps a batch on the device refuses, or shares less in, without a device: places that end while others still read their pages."""
import numpy as np
import pytest

from mycaffe_amd.layers import PagedBatch
from tests.test_layers_batch import Memory


def batch_of(*lens, tokens=50):
    cuda = Memory()
    batch = PagedBatch(cuda, len(lens), tokens, 64, 4, 16)
    batch.lens.mutable_cpu_data = np.array(lens, np.float32)
    return cuda, batch


def test_a_lender_ends_last():
    cuda, batch = batch_of(20, 0, 0)
    batch.Begin({1: (0, 8)})
    kept = batch.new.mutable_cpu_data.copy()
    for new in ([-1, 3, 0], [-1, 0, 0], [-1, 3, 5], [-5, 0, 0]):     # in the step in which the other one begins, before it has, ...
        with pytest.raises(ValueError, match="place 0 .* place 1"):
            batch.Step(new)
        assert cuda.calls.count("PagedPlan") == 0 and np.array_equal(batch.new.mutable_cpu_data, kept)
    batch.Step([1, 3, 0])
    with pytest.raises(ValueError, match="place 0 .* place 1"):           # ... and while it lasts
        batch.Step([-1, 1, 0])
    assert cuda.calls.count("PagedPlan") == 1
    batch.Step([1, -1, 0])
    batch.Step([-1, 1, 0])
    assert cuda.calls.count("PagedPlan") == 3


def test_both_end_at_once():
    cuda, batch = batch_of(20, 0, 0)
    batch.Begin({1: (0, 8), 2: (0, 4)})
    batch.Step([1, 3, 3])
    with pytest.raises(ValueError, match="place 0 .* place 2"):
        batch.Step([-1, -1, 1])
    batch.Step([-1, -1, -1])
    assert cuda.calls.count("PagedPlan") == 2


def test_one_behind_the_other():
    """The third begins in pages of the second, the first of which are the first's: it keeps the second, which keeps the first."""
    cuda, batch = batch_of(20, 0, 0)
    batch.Begin({1: (0, 8)})
    batch.Step([1, 10, 0])
    batch.Begin({2: (1, 16)})
    batch.Step([1, 1, 3])
    for new in ([-1, 1, 1], [1, -1, 1], [-1, -1, 1]):
        with pytest.raises(ValueError):
            batch.Step(new)
    batch.Step([1, -1, -1])
    batch.Step([-1, 0, 0])


def test_what_a_step_without_an_argument_ended():
    """Its numbers are the device's, so what is borrowed is looked up there before a step is refused."""
    cuda, batch = batch_of(20, 0, 0)
    batch.Begin({1: (0, 8)})
    batch.Step([1, 3, 0])
    batch.Step()
    batch.shared.mutable_cpu_data = np.zeros(3, np.float32)              # what the plan writes of a place that ended
    batch.Step([-1, 0, 0])
    assert cuda.calls.count("PagedPlan") == 3


def test_groups_of_places_that_hold_others_now():
    cuda, batch = batch_of(20, 30, 30, 40, 40)
    said = lambda: (batch.nGroups, list(batch.bounds.mutable_cpu_data), list(batch.common.mutable_cpu_data))  # noqa: E731
    batch.Share([0, 3, 5], [16, 8])
    batch.Step([1, -1, 1, 1, 1])
    batch.Step([1, 0, 1, 1, 1])
    assert said() == (2, [0, 3, 5], [16, 8])              # nothing in place 1: what the others share they still do
    batch.Step([1, 7, 1, 1, 1])
    assert said() == (2, [0, 3, 5], [0, 8])               # another sequence there: its first positions are its own
    batch.Step([1, 1, 1, -1, 1])
    batch.Step([1, 1, 1, 2, 1])
    assert batch.nGroups == 0                             # nobody shares anything
    batch.Share([0, 1, 3], [0, 16])
    batch.Step([-1, 1, 1, 1, 1])
    batch.Step([4, 1, 1, 1, 1])
    assert said() == (2, [0, 1, 3], [0, 16])              # place 0 is in no group that shares


def test_groups_said_again_count():
    cuda, batch = batch_of(20, 0, 30)
    batch.Share([0, 3], [16])
    batch.Step([1, -1, 1])
    batch.Begin({1: (0, 16)})
    batch.Share([0, 3], [16])
    batch.Step([1, 5, 1])
    batch.Step([1, 1, 1])
    assert batch.nGroups == 1 and list(batch.common.mutable_cpu_data) == [16]
    batch.Share()
    batch.Step([1, -1, 1])
    batch.Step([1, 2, 1])
    assert batch.nGroups == 0


@pytest.mark.parametrize("rows,pages,page,width,most", [(50, 64, 4, 16, 50), (200, 64, 4, 16, 64), (200, 9, 4, 16, 36)])
def test_wishes_that_no_step_can_grant(rows, pages, page, width, most):
    """They would wait for ever, and all places behind them."""
    cuda = Memory()
    batch = PagedBatch(cuda, 3, rows, pages, page, width)
    kept = batch.new.mutable_cpu_data.copy()
    for wish in (most + 1, 1e9, np.inf, np.nan, 0.5, -0.5):
        with pytest.raises(ValueError, match="up to %d " % most):
            batch.Step([1, wish, 1])
        assert cuda.calls.count("PagedPlan") == 0 and np.array_equal(batch.new.mutable_cpu_data, kept)
    batch.Step([1, most, 1])
    batch.Step([-1, -3, 0])
    assert cuda.calls.count("PagedPlan") == 2
