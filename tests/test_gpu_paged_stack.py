"""The stack of free pages that PAGED_PLAN (csrc/paged_plan.hip) leaves, all of it: up to its number the loop's, behind it what was there."""
import numpy as np
import pytest

from mycaffe_amd.cudadnn import CudaDnn, CudaDnnDouble
from oracle import serving_ref as S
from tests.test_gpu_paged_plan import Call, state

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[CudaDnn, CudaDnnDouble])
def cuda(request):
    c = request.param(0)
    yield c
    c.Dispose()


def check(cuda, new, lens, table, free, tokens, page, origin=None, shared=None):
    """In place and elsewhere; what the loop says."""
    B, W = table.shape
    want = S.plan(new, lens, table, free, tokens, page, origin, shared)
    n = int(want["free"][0])
    for place in (False, True):
        c = Call(cuda, new, lens, table, free, tokens, page, origin, shared, place=place)
        c()
        c.check(want, B, W)
        got = c.get("free_out")
        assert got[0] == n and np.array_equal(got[1:1 + n], want["free"][1:1 + n])
        assert np.array_equal(got[1 + n:], np.asarray(free, np.float64)[1 + n:] if place else np.full(len(free) - 1 - n, -5.0)), "entries behind the number are left alone"
        c.close()
    return want


# sequences, width of their tables, positions of a page: lists of one look and of several, batches of one list and of several
SIZES = [(1, 4, 4), (5, 6, 4), (16, 100, 2), (17, 12, 4), (64, 200, 4), (1024, 3, 8), (1025, 6, 8), (2100, 9, 3)]


@pytest.mark.parametrize("B,W,page", SIZES)
def test_what_remains(cuda, B, W, page):
    # by turns: nothing ends; more is taken than comes back; more comes back than is taken; nothing grows; the stack is empty
    for seed, (ends, begins, spare, most) in enumerate([(0.0, 0.3, 3 * B, W * page // 2 + 1), (0.2, 0.5, B * W, W * page // 2 + 1), (0.6, 0.1, B, 2), (0.9, 0.0, 2, 1), (0.4, 0.4, 0, W * page // 2 + 1)]):
        rng = np.random.default_rng(seed)
        new, lens, table, free = state(rng, B, W, page, spare, ends, begins, 0.1, most)
        if seed == 3:
            new = np.minimum(new, 0)
        check(cuda, new, lens, table, free, int(max(1, np.maximum(new, 0).sum())), page)


@pytest.mark.parametrize("B,W,page", [(5, 6, 4), (64, 200, 4), (2100, 9, 3)])
def test_pages_that_come_back_and_go_again(cuda, B, W, page):
    """Rows with holes end, borrowed pages stay with their owners, and all that comes back is taken again in the same call."""
    rng = np.random.default_rng(B)
    new, lens, table, free = state(rng, B, W, page, 0, 0.5, 0.4, 0.0, W * page)
    table[(rng.random(table.shape) < 0.2) & (new < 0)[:, None]] = -1
    shared = np.where(lens > 0, np.minimum(rng.integers(0, 3, B) * page, lens // page * page), 0).astype(float)
    want = check(cuda, new, lens, table, free, int(max(1, np.maximum(new, 0).sum())), page, np.full(B, -1.0), shared)
    # most of it, until the first one waits
    assert B < 64 or want["free"][0] <= W


def test_a_long_stack(cuda):
    """Most of it remains whatever a call decides, and is copied beside the decisions."""
    rng = np.random.default_rng(1)
    for B, tokens, spare in ((20, 40, 70000), (3, 9, 5000), (40, 20000, 12000)):
        new, lens, table, free = state(rng, B, 30, 16, spare, 0.2, 0.3, 0.1, max(1, tokens // B))
        check(cuda, new, lens, table, free, tokens, 16)


def test_a_stack_that_is_full(cuda):
    """Pages of the rows that end for which there is no room on it are dropped, as the loop does."""
    table = np.array([[0, 1, 2], [3, 4, -1], [-1, -1, -1]], float)
    for new in ([-1, -1, 0], [-1, -1, 5], [-1, -1, 13]):
        check(cuda, np.array(new, float), np.array([12.0, 8.0, 0.0]), table, np.array([5, 7, 6, 5, 4, 3, 9, 9, 9], float), 16, 4)
