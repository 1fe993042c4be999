"""Paged caches and norms of heads where sizes end: starts that decrease, 2^24 tokens, rows beyond one axis of a launch, no scratch memory, two kernel
objects at once, pages that sequences share."""
import numpy as np
import pytest

from mycaffe_amd.cudadnn import CudaDnnDouble
from tests.conftest import Dev
from tests.test_gpu_paged import Cache, TYPES, attention, check_attention, rounded

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act16", [False, True])
@pytest.mark.parametrize("tokens", [2000, 4000])       # single tokens by the split of positions, chunks
def test_lists_of_work_that_are_none(dev, tokens, act16):
    """Starts that decrease give the same tokens to many sequences, more units of work than are counted: nothing is written, and the next call is right."""
    kvH, hs, page, width, batch = 8, 64, 1024, 256, 2000
    k, table = dev.zeros(4 * kvH * page * hs, act16), dev.zeros(batch * width)
    starts = np.zeros(batch + 1, np.float32)
    starts[1::2] = tokens
    hs_, hl = dev.put(starts), dev.put(np.full(batch, width * page, np.float32))
    q, y = dev.zeros(tokens * kvH * hs, act16), dev.put(np.full(tokens * kvH * hs, 7.0, np.float32), act16)
    dev.cuda.AttnPagedForward(batch, tokens, kvH, kvH, hs, 4, page, width, q, k, k, table, hs_, hl, y, kvH * page * hs, page * hs, hs)
    assert (dev.get(y, (tokens * kvH * hs,)) == 7.0).all()
    rng = np.random.default_rng(30)
    check_attention(dev, rng, Cache(dev, rng, [(1, 300, 0), (1, 40, 0), (30, 95, 16)], 2, hs, 16, "pos", act16), 4, act16)


def test_starts_that_decrease_a_little(dev):
    """A list that can be counted: tokens of several sequences get the result of one of them, rows behind stay as they were."""
    rng = np.random.default_rng(31)
    kvH, hs, page, N = 4, 64, 16, 3000
    k, v = (dev.put(rounded(rng.standard_normal(8 * kvH * page * hs), True), True) for _ in range(2))
    q, y = dev.put(rounded(rng.standard_normal(N * kvH * hs), True), True), dev.put(np.full(N * kvH * hs, 7.0, np.float32), True)
    starts, lens, table = dev.put(np.float32([0, 2900, 0, 2900])), dev.put(np.float32([64, 64, 64])), dev.put(np.tile(np.float32([5, 1, 7, 2]), 3))
    dev.cuda.AttnPagedForward(3, N, kvH, kvH, hs, 8, page, 4, q, k, v, table, starts, lens, y, kvH * page * hs, page * hs, hs)
    got = dev.get(y, (N, kvH * hs))
    assert np.isfinite(got).all() and (got[2900:] == 7.0).all()
    assert (got[:2900 - 64] == 0).all() and (got[2900 - 64:2900] != 0).any()


@pytest.mark.parametrize("hs", [2, 4])       # the plain kernel, the split of positions
def test_as_many_tokens_as_there_can_be(dev, hs):
    """2^24 tokens, of which the last three have positions."""
    N, rng = 1 << 24, np.random.default_rng(32)
    k, v = np.float32(rng.standard_normal((2, 3, hs)))
    hk, hv = (dev.put(np.concatenate([a, np.full((5, hs), np.nan, np.float32)])) for a in (k, v))
    q = np.zeros((N, hs), np.float32)
    q[-3:] = rng.standard_normal((3, hs))
    hq, hy = dev.put(q), dev.zeros(N * hs)
    dev.cuda.set(N * hs, hy, 7.0)
    dev.cuda.AttnPagedForward(1, N, 1, 1, hs, 1, 8, 1, hq, hk, hv, dev.put(np.float32([0])), dev.put(np.float32([0, N])), dev.put(np.float32([3])), hy, 8 * hs, 8 * hs, hs)
    got = dev.get(hy, (N, hs))
    assert not got[:-3].any()
    c = type("C", (), dict(kvH=1, hs=hs, tokens=3, seqs=[(3, 3, 0)], dense=[(k[:, None], v[:, None])]))
    want, tol = attention(c, q[-3:, None], 1, False, None, False)
    assert (abs(got[-3:, None] - want) <= tol).all()


def test_as_many_tokens_as_there_can_be_in_double():
    cuda, N = CudaDnnDouble(0), 1 << 24
    try:
        put = lambda a: cuda.AllocMemory(np.asarray(a, np.float64))
        qkv = np.zeros((N, 6))
        qkv[-1] = [1, 2, 3, 4, 5, 6]
        hx, hq, hy, hk, hv = put(qkv), put(np.full(2 * N, 7.0)), put(np.full(2 * N, 7.0)), put(np.full(4, 7.0)), put(np.full(4, 7.0))
        where = (1, N, 1, 1, 2, 1, 2, 1)
        meta = (put([0.0]), put([0.0, N]), put([1.0]))
        cuda.PagedAppend(*where, hx, hq, hk, hv, *meta, 4, 4, 2)
        cuda.AttnPagedForward(*where, hq, hk, hv, *meta, hy, 4, 4, 2)
        q, y = (np.asarray(cuda.GetMemoryFloat(h)).reshape(N, 2) for h in (hq, hy))
        assert np.array_equal(q, qkv[:, :2]) and np.array_equal(y[-1], [5, 6]) and not y[:-1].any()
        assert np.array_equal(cuda.GetMemoryFloat(hk), [3, 4, 7, 7]) and np.array_equal(cuda.GetMemoryFloat(hv), [5, 6, 7, 7])
    finally:
        cuda.Dispose()


def test_norms_of_more_rows_than_an_axis_has(dev):
    """2^29 + 11 positions, in place: every row of (3, 3) becomes (1, 1) / sqrt(1 + eps / 9), in 16 bits (1, 1)."""
    cuda, T = dev.cuda, (1 << 29) + 11
    q, k = cuda.AllocMemory(2 * T, bHalfSize=True), cuda.AllocMemory(2 * T, bHalfSize=True)
    try:
        for h in (q, k):
            cuda.set(2 * T, h, 3.0)
        cuda.QkNormRopeForward(1, T, 1, 1, 2, q, k, 0, 0, q, k)
        for h in (q, k):
            for at in (0, (1 << 28) - 4, 1 << 29, 2 * ((1 << 28) - 4), 2 * T - 8):
                view = cuda.CreateMemoryPointer(h, at, 8)
                assert (np.asarray(dev.get(view, (8,))) == 1.0).all(), at
                cuda.FreeMemoryPointer(view)
    finally:
        cuda.FreeMemory(q)
        cuda.FreeMemory(k)


@pytest.mark.parametrize("act16,cache16", TYPES)
def test_without_scratch_memory(monkeypatch, act16, cache16):
    monkeypatch.setenv("MYCAFFE_HIP_SCRATCH_LIMIT", "1000000")
    dev, rng = Dev(), np.random.default_rng(33)
    try:
        check_attention(dev, rng, Cache(dev, rng, [(1, 300, 0), (40, 95, 16), (0, 3, 0), (2, 1, 0)], 2, 64, 16, "pos", cache16), 4, act16)
    finally:
        dev.close()


@pytest.mark.parametrize("act16,cache16", TYPES)
def test_pages_that_sequences_share(dev, act16, cache16):
    """Four sequences that begin with the same pages, as prompts with a common beginning do."""
    rng = np.random.default_rng(34)
    c = Cache(dev, rng, [(1, 100, 0), (30, 100, 0), (1, 70, 0), (5, 90, 0)], 2, 64, 16, "head", cache16)
    shared = 4
    for b in range(1, 4):
        c.table[b, :shared] = c.table[0, :shared]
        for mine, first in zip(c.dense[b], c.dense[0]):
            mine[:16 * shared] = first[:16 * shared]
    c.h["table"] = dev.put(c.table)
    check_attention(dev, rng, c, 4, act16)


def test_two_kernel_objects_at_once():
    """Calls of two streams in flight together, each with its own lists, partial results and tickets."""
    devs = [Dev(), Dev()]
    try:
        rng, H = np.random.default_rng(35), 8
        work = []
        for i, dev in enumerate(devs):
            for act16, seqs in ((True, [(1, 900 + 50 * b, 0) for b in range(12)]), (False, [(70, 300, 0), (1, 900, 0)]), (True, [(400, 500, 0), (9, 800, 0)])):
                c = Cache(dev, rng, seqs, 2, 64, 16, "pos", act16)
                q = rounded(rng.standard_normal((c.tokens, H, 64)), act16)
                work.append((i, c, q, act16, dev.put(q, act16), dev.zeros(q.size, act16)))
        for _ in range(5):
            for i, c, q, act16, hq, hy in sorted(work, key=lambda w: w[1].tokens):
                c.attend(hq, hy, H)
        for i, c, q, act16, hq, hy in work:
            want, tol = attention(c, q, H, act16, None, act16)
            assert (abs(devs[i].get(hy, q.shape) - want) <= tol).all()
    finally:
        for dev in devs:
            dev.close()


WIDE = [
    # heads of more than 128 values, and sizes and strides that are read value by value
    ("one", 1, 1, 256, 16, "head", [(1, 1, 0)], 0),
    ("long", 4, 2, 256, 64, "head", [(1, 9000, 0), (1, 700, 0)], 0),
    ("groups_of_seven", 7, 1, 200, 8, "pos", [(1, 70, 0), (3, 9, 0), (0, 5, 0)], 2),
    ("chunks", 4, 2, 136, 24, "head", [(40, 40, 0), (70, 300, 0), (1, 33, 0), (17, 90, 16)], 5),
    ("heads_of_two_tiles", 20, 1, 192, 16, "pos", [(1, 200, 0), (9, 60, 0)], 0),
    ("many", 2, 1, 256, 8, "head", [(b % 3, b % 3 + 7 * b % 61, 0) for b in range(300)], 1),
    ("plain_one", 2, 1, 198, 16, "head", [(1, 1, 0), (1, 900, 0)], 0),
    ("plain_chunks", 6, 3, 46, 16, "pos", [(60, 90, 0), (50, 333, 32), (0, 9, 0), (1, 40, 0), (3, 2, 0)], 3),
    ("plain_wide", 4, 4, 254, 7, "head", [(70, 100, 0), (65, 65, 0)], 0),
]


@pytest.mark.parametrize("act16,cache16", TYPES)
@pytest.mark.parametrize("name,H,kvH,hs,page,order,seqs,pad", WIDE, ids=[s[0] for s in WIDE])
def test_wide_and_odd_heads(dev, name, H, kvH, hs, page, order, seqs, pad, act16, cache16):
    rng = np.random.default_rng(36 + hs)
    c = Cache(dev, rng, seqs, kvH, hs, page, order, cache16, pad=pad)
    q = rounded(rng.standard_normal((c.tokens, H, hs)) * 1.5, act16)
    hq, hy = dev.put(q, act16), dev.put(np.full(q.size, 7.0, np.float32), act16)
    c.attend(hq, hy, H)
    got = dev.get(hy, q.shape)
    c.attend(hq, hy, H)
    assert np.array_equal(got, dev.get(hy, q.shape), equal_nan=True)      # the same bits every time
    want, tol = attention(c, q, H, act16, None, act16)
    for b, (n, _, gone) in enumerate(seqs):
        rows = slice(int(c.starts[b]), int(c.starts[b]) + n)
        # only whole pages are given up: NaN in what is left of one is seen
        assert np.isnan(got[rows]).all() if gone % page else (abs(got[rows] - want[rows]) <= tol[rows]).all(), b
    assert (got[int(c.starts[-1]):] == 7.0).all()


@pytest.mark.parametrize("act16,cache16", TYPES)
@pytest.mark.parametrize("hs", [46, 254, 256])
def test_wide_and_odd_heads_with_values_that_are_not_finite(dev, hs, act16, cache16):
    """What later tokens have written - keys and values of infinity and NaN - has no say in the tokens before them."""
    rng = np.random.default_rng(37)
    c = Cache(dev, rng, [(12, 50, 0), (1, 30, 0)], 2, hs, 16, "head", cache16)
    q = rounded(rng.standard_normal((c.tokens, 4, hs)), act16)
    hq, hy = dev.put(q, act16), dev.zeros(q.size, act16)
    want, tol = attention(c, q, 4, act16, None, act16)
    k, v = c.get("k").copy(), c.get("v").copy()
    for t, bad in ((44, np.nan), (45, np.inf), (49, -np.inf)):       # tokens 6, 7 and 11 of the first sequence
        page = int(c.table[0, t // 16])
        k[page, :, t % 16, 3], v[page, :, t % 16, 5] = bad, bad
    c.h["k"], c.h["v"] = dev.put(c.laid(k), cache16), dev.put(c.laid(v), cache16)
    c.attend(hq, hy, 4)
    got = dev.get(hy, q.shape)
    clean = [0, 1, 2, 3, 4, 5, 12]
    assert (abs(got[clean] - want[clean]) <= tol[clean]).all()
    assert np.isnan(got[6:12, :, 5]).all()


MANY = [
    # more sequences than one scan has threads, chunks and single tokens among each other
    ("chunks", 4, 2, 64, 16, [(1 if b % 3 else 20 + b % 17, 40 + 13 * b % 90, 0) for b in range(600)], (True, False)),
    ("long_chunks_64", 8, 1, 64, 16, [(1 if b % 29 == 0 else 40 + b % 5, 60 + b % 50, 16 * (b % 2)) for b in range(300)], (True,)),
    ("long_chunks_128", 8, 1, 128, 32, [(1 if b % 29 == 0 else 40 + b % 5, 60 + b % 50, 0) for b in range(300)], (True,)),
]


@pytest.mark.parametrize("name,H,kvH,hs,page,seqs,types", MANY, ids=[m[0] for m in MANY])
def test_more_chunks_than_a_scan(dev, name, H, kvH, hs, page, seqs, types):
    for act16 in types:
        rng = np.random.default_rng(38)
        check_attention(dev, rng, Cache(dev, rng, seqs, kvH, hs, page, "head", act16, pad=3), H, act16)
