"""What the layers do for a batch of sequences on the device, and what they refuse, without one."""
import numpy as np
import pytest

from mycaffe_amd.layers import Blob, PagedBatch, PagedSequences
from tests.test_layers_kept import Context
from tests.test_layers_paged import attention, serve


class Memory(Context):
    """A stand-in context that keeps what is written."""

    def __init__(self):
        super().__init__()
        self.kept = {}

    def SetMemory(self, h, values, *a, **k):
        self.kept[h] = np.array(values).reshape(-1)

    def GetMemoryFloat(self, h, *a, **k):
        return self.kept[h]


def test_a_pass_takes_the_attention_of_its_groups():
    cuda = Memory()
    batch, layer = PagedBatch(cuda, 4, 7, 6, 4, 4), attention(cuda)
    batch.Step([2, 1, 0, 1])
    assert cuda.calls.count("PagedPlan") == 1
    serve(cuda, [layer], batch)
    batch.Share([0, 2, 4], [4, 8])
    assert batch.nGroups == 2
    serve(cuda, [layer], batch)
    batch.Share()
    batch.Step()
    serve(cuda, [layer], batch)
    assert [c for c in cuda.calls if c.startswith("AttnPaged")] == ["AttnPagedForward", "AttnPagedPrefixForward", "AttnPagedForward"]
    with pytest.raises(ValueError):
        layer.ForwardPaged(Blob(cuda, (1, 6, 16)), batch, Blob(cuda))


def test_state_at_the_begin():
    cuda = Memory()
    batch = PagedBatch(cuda, 3, 8, 5, 4, 2)
    assert list(batch.free.mutable_cpu_data) == [5, 4, 3, 2, 1, 0] and not batch.lens.mutable_cpu_data.any()
    assert (batch.table.mutable_cpu_data == -1).all() and (batch.origin.mutable_cpu_data == -1).all()
    batch.Begin({1: (0, 8), 2: (0, 4)})
    assert list(batch.origin.mutable_cpu_data) == [-1, 0, 0] and list(batch.shared.mutable_cpu_data) == [0, 8, 4]


def test_refusals():
    cuda = Memory()
    batch = PagedBatch(cuda, 3, 8, 5, 4, 2)
    for new in ([1, 1], [1, 1, 1, 1], 1, [[1, 1, 1]]):
        with pytest.raises(ValueError):
            batch.Step(new)
    for places in ({3: (0, 4)}, {0: (3, 4)}, {-1: (0, 4)}, {1: (1, 4)}):
        with pytest.raises(ValueError):
            batch.Begin(places)
    batch.lens.mutable_cpu_data = np.array([4, 0, 0])
    with pytest.raises(ValueError):
        batch.Begin({0: (1, 4)})
    for bounds, positions in (([0, 2], [4, 4]), ([0, 2, 1], [4, 4]), ([0, 4], [4]), ([-1, 3], [4]), ([], [4])):
        with pytest.raises(ValueError):
            batch.Share(bounds, positions)
        assert batch.nGroups == 0
    number = Blob(cuda, (3,))
    for logits, random, heat in (((1, 7, 9), (3,), None), ((1, 8, 9), (2,), None), ((1, 8, 9), (3,), Blob(cuda, (8,)))):
        with pytest.raises(ValueError):
            batch.Sample(Blob(cuda, logits), Blob(cuda, random), heat)
    batch.Sample(Blob(cuda, (1, 8, 9)), number, number, None, number)
    assert cuda.calls.count("SampleForward") == 1 and cuda.calls.count("PagedPlan") == 0


@pytest.mark.parametrize("kind", [PagedBatch, PagedSequences])
def test_everything_is_given_back(kind):
    cuda = Memory()
    paged = PagedBatch(cuda, 2, 3, 6, 4, 4) if kind is PagedBatch else PagedSequences(cuda, 6, 4, 4)
    layer = attention(cuda)
    if kind is PagedBatch:
        paged.Share([0, 2], [4])
        paged.Step([2, 1])
    else:
        paged.Step({"a": 2, "b": 1})
    held = set(cuda.live)
    k, v = paged.Cache(layer, 2, 8, False)
    rope = paged.Rope(2, 8, 10000.0)
    assert {k.gpu_data, v.gpu_data, rope} == set(cuda.live) - held
    paged.Dispose()
    assert not [h for h in (k.gpu_data, v.gpu_data, rope) if h in cuda.live]
    paged.Dispose()
