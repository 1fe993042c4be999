"""PAGED_PLAN (csrc/paged_plan.hip) against a plain loop over the sequences: every number it writes, whole ones, has to be the loop's."""
import numpy as np
import pytest

from mycaffe_amd.cudadnn import CudaDnn, CudaDnnDouble, CudaDnnError
from oracle import serving_ref as S

pytestmark = pytest.mark.gpu


def state(rng, B, W, page, spare, ends=0.1, begins=0.1, idle=0.1, most=1, fill=0.6):
    """Sequences of all lengths in pages of any order, wishes of all kinds."""
    kind = rng.random(B)
    lens = np.minimum(1 + (W * page * fill * rng.random(B)).astype(int), W * page)
    new = 1 + (most * rng.random(B)).astype(int) if most > 1 else np.ones(B, int)
    begin = kind < begins
    lens[begin] = 0
    new[(kind >= begins) & (kind < begins + ends)] = -1
    new[(kind >= begins + ends) & (kind < begins + ends + idle)] = 0
    held = -(-lens // page)
    pages = int(held.sum()) + spare + 2
    order = rng.permutation(pages)
    table = np.full((B, W), -1.0)
    at = 0
    for b in range(B):
        table[b, :held[b]] = order[at:at + held[b]]
        at += held[b]
    free = np.full(pages + 1, -7.0)
    free[0], free[1:1 + spare] = spare, order[at:at + spare]
    return new.astype(float), lens.astype(float), table, free


class Call:
    """One call on device memory; in place or not, with lenders or not."""

    def __init__(self, cuda, new, lens, table, free, tokens, page, origin=None, shared=None, place=False, rows=True, filler=-5.0):
        self.cuda, (B, W), self.h = cuda, table.shape, {}
        self.tokens, self.place, self.rows = tokens, place, rows
        put = lambda n, v: self.h.__setitem__(n, cuda.AllocMemory(np.asarray(v, cuda.DTYPE).reshape(-1)))  # noqa: E731
        for n, v in (("new", new), ("lens", lens), ("table", table), ("free", free)):
            put(n, v)
        if shared is not None:
            put("origin", origin)
            put("shared", shared)
        for n, v in (("lens", lens), ("table", table), ("free", free)) + ((("shared", shared),) if shared is not None else ()):
            if place:
                self.h[n + "_out"] = self.h[n]
            else:
                put(n + "_out", np.full(np.size(v), filler))
        for n, count in (("starts", B + 1), ("positions", tokens), ("slots", tokens), ("last", B)):
            put(n, np.full(count, filler))
        self.args = [B, tokens, len(free) - 1, page, W]

    def __call__(self):
        h = self.h
        more = [h["origin"], h["shared"], h["shared_out"]] if "shared" in h else []
        rows = [h["positions"], h["slots"]] if self.rows else [0, 0]
        self.cuda.PagedPlan(*self.args, h["new"], h["lens"], h["table"], h["free"], h["lens_out"], h["table_out"], h["free_out"], h["starts"], *rows, h["last"], *more)

    def get(self, name):
        return np.asarray(self.cuda.GetMemoryFloat(self.h[name]), np.float64)

    def check(self, want, B, W):
        n = want["starts"][-1]
        assert np.array_equal(self.get("starts"), want["starts"])
        assert np.array_equal(self.get("last"), want["last"])
        assert np.array_equal(self.get("lens_out"), want["lens"])
        assert np.array_equal(self.get("table_out").reshape(B, W), want["table"])
        free = self.get("free_out")
        assert free[0] == want["free"][0]
        listed = want["listed"]
        assert np.array_equal(free[1:1 + listed], want["free"][1:1 + listed])
        if self.rows:
            for name in ("positions", "slots"):
                got = self.get(name)
                assert np.array_equal(got[:n], want[name])
                assert np.all(got[n:] == -5.0), "rows behind the last sequence are left alone"
        if "shared_out" in self.h:
            assert np.array_equal(self.get("shared_out"), want["shared"])

    def close(self):
        for h in set(self.h.values()):
            self.cuda.FreeMemory(h)


@pytest.fixture(params=[CudaDnn, CudaDnnDouble])
def cuda(request):
    c = request.param(0)
    yield c
    c.Dispose()


SIZES = [(1, 1, 1), (1, 8, 16), (3, 5, 7), (16, 12, 4), (17, 12, 4), (16, 64, 32), (64, 16, 16), (65, 9, 24), (1000, 4, 8), (1024, 3, 8), (1025, 6, 8), (2100, 5, 3)]


@pytest.mark.parametrize("place", [False, True])
@pytest.mark.parametrize("B,W,page", SIZES)
def test_steps_against_the_loop(cuda, B, W, page, place):
    for seed, (most, ends, begins, spare) in enumerate([(1, 0.0, 0.0, B + 1), (1, 0.2, 0.2, 2 * B), (W * page // 2 + 1, 0.1, 0.5, B * W), (5, 0.3, 0.3, B // 3)]):
        rng = np.random.default_rng(seed)
        new, lens, table, free = state(rng, B, W, page, spare, ends, begins, 0.1, most)
        tokens = int(max(1, np.maximum(new, 0).sum() * (1.0 if seed < 3 else 0.8)))
        want = S.plan(new, lens, table, free, tokens, page)
        c = Call(cuda, new, lens, table, free, tokens, page, place=place)
        c()
        c.check(want, B, W)
        c.close()


@pytest.mark.parametrize("place", [False, True])
@pytest.mark.parametrize("B,W,page", [(3, 5, 7), (64, 16, 16), (1500, 6, 8)])
def test_sequences_that_begin_behind_another_ones_prompt(cuda, B, W, page, place):
    rng = np.random.default_rng(B)
    new, lens, table, free = state(rng, B, W, page, 2 * B, 0.2, 0.4, 0.1, page)
    origin = rng.integers(-1, B + 1, B).astype(float)
    origin[::7] = np.arange(B)[::7]                        # itself: nothing to borrow
    # of sequences that go on, what they hold of others; a sequence that ends keeps these pages out of the stack
    shared = np.floor(rng.random(B) * W * page * 1.2)
    shared[lens > 0] = np.minimum(shared, lens)[lens > 0] // page * page
    tokens = int(np.maximum(new, 0).sum() * 0.9)
    want = S.plan(new, lens, table, free, tokens, page, origin, shared)
    c = Call(cuda, new, lens, table, free, tokens, page, origin, shared, place=place)
    c()
    c.check(want, B, W)
    c.close()


def test_a_large_step_is_written_by_its_own_launch(cuda):
    """Rows beyond what the first workgroup writes, and positions without slots."""
    B, W, page = 90, 40, 16
    rng = np.random.default_rng(2)
    new, lens, table, free = state(rng, B, W, page, B * W, 0.0, 0.9, 0.0, W * page, fill=0.0)
    new = np.where(lens == 0, new, 1)
    tokens = int(new.sum())
    assert tokens > 16384
    want = S.plan(new, lens, table, free, tokens, page)
    for rows in (True, False):
        c = Call(cuda, new, lens, table, free, tokens, page, rows=rows)
        c()
        c.check(want, B, W)
        c.close()


def test_numbers_out_of_range(cuda):
    """Lengths, wishes, stacks and entries that are no such numbers are brought into their range."""
    B, W, page = 8, 4, 4
    nan = float("nan")
    table = np.array([[0, 1, nan, -1], [2, 99, -3, 3], [4, 5, 6, 7], [-1] * 4, [8, 9, -1, -1], [10, -1, -1, -1], [-1] * 4, [-1] * 4], float)
    new = np.array([1, -2.5, 5, nan, 0.5, 1e30, 2, -0.5])
    lens = np.array([7, 1e9, 16, nan, 8, 3, -4, 0])
    free = np.array([3, 11, nan, 55, 12, 13, 14, 15, 16, 17, 18, 19, 20], float)
    for count in (3, nan, -2, 1e9, 12):
        free[0] = count
        want = S.plan(new, lens, table, free, 100, page)
        for place in (False, True):
            c = Call(cuda, new, lens, table, free, 100, page, place=place)
            c()
            for name in ("lens", "starts", "last"):
                assert np.array_equal(c.get(name + "_out" if name == "lens" else name), want[name]), (count, name)
            assert np.array_equal(c.get("table_out").reshape(B, W), want["table"], equal_nan=True), count
            assert c.get("free_out")[0] == want["free"][0]
            c.close()


def test_steps_in_place_one_after_the_other(cuda):
    """A server's life: sequences begin, grow, end and begin again in place; at any time every page belongs to one sequence or to the stack."""
    B, W, page, pages = 70, 6, 8, 150
    rng = np.random.default_rng(9)
    lens, table, free = np.zeros(B), np.full((B, W), -1.0), np.concatenate([[pages], rng.permutation(pages)]).astype(float)
    c = Call(cuda, np.zeros(B), lens, table, free, 300, page, place=True)
    for step in range(25):
        new = np.where(lens == 0, (rng.random(B) < 0.3) * (1 + rng.integers(0, 20, B)), np.where(rng.random(B) < 0.1, -1, 1)).astype(float)
        want = S.plan(new, lens, table, free, 300, page)
        c.cuda.SetMemory(c.h["new"], np.asarray(new, c.cuda.DTYPE))
        c()
        lens, table, free = np.asarray(want["lens"], float), want["table"], want["free"]
        assert np.array_equal(c.get("lens"), lens) and np.array_equal(c.get("table").reshape(B, W), table)
        got = c.get("free")
        n = int(free[0])
        assert got[0] == n and np.array_equal(got[1:1 + n], free[1:1 + n])
        held = table[table >= 0]
        assert sorted(np.concatenate([held, free[1:1 + n]]).tolist()) == list(range(pages))
    c.close()


def test_refusals(cuda):
    rng = np.random.default_rng(0)
    new, lens, table, free = state(rng, 4, 3, 4, 8)
    c = Call(cuda, new, lens, table, free, 16, 4, np.zeros(4), np.zeros(4))
    h, a = c.h, c.args
    good = [h[n] for n in ("new", "lens", "table", "free", "lens_out", "table_out", "free_out", "starts", "positions", "slots", "last", "origin", "shared", "shared_out")]

    def refused(sizes=None, **change):
        v = list(good)
        for i, x in change.items():
            v[int(i[1:])] = x
        with pytest.raises(CudaDnnError):
            cuda.PagedPlan(*(sizes or a), *v)

    for i in range(5):
        for bad in (0, -1, (1 << 24) + 1):
            refused(a[:i] + [bad] + a[i + 1:])
    refused([4, 16, 1 << 22, 8, 3])                      # slots beyond 2^24
    refused([4, 16, len(free) - 1, 1 << 20, 3 << 8])     # positions beyond 2^24
    refused([5] + a[1:])                                 # memory too small
    refused(_4=h["lens"])                                # lengths in place, the table elsewhere
    refused(_13=h["shared"])
    refused(_7=h["new"])                                 # outputs over inputs, and over each other
    refused(_8=h["slots"])
    refused(_10=h["lens_out"])
    refused(_11=0)                                       # all three of what is borrowed, or none
    refused(_12=0)
    refused(_13=0)
    for i in (0, 1, 2, 3, 4, 5, 6, 7, 10):
        refused(**{"_%d" % i: 0})
    if cuda.DTYPE == np.float32:
        half = cuda.AllocMemory(64, bHalfSize=True)
        for i in range(14):
            refused(**{"_%d" % i: half})
        cuda.FreeMemory(half)
    cuda.PagedPlan(*a, *good)
    c.close()
