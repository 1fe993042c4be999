"""Paged caches: new tokens appended (id 2015) and attention over the pages (id 2016), against the definitions in 64 bits.

Whatever no token may see is NaN in these caches: positions behind a sequence, pages that are nobody's.  Tolerances count roundings: u is half a
step of a type (finfo.eps / 2); fp32 sums of n terms are off by at most n u of the sum of their magnitudes."""
import numpy as np
import pytest

from tests.conftest import bf16_round
from mycaffe_amd.cudadnn import CudaDnnError

pytestmark = pytest.mark.gpu

U32, U16 = 2.0 ** -24, 2.0 ** -8
EPS, THETA = 1e-5, 10000.0


def rounded(a, half):
    return bf16_round(a) if half else np.float32(a)


class Cache:
    """Pages of sequences [(new tokens, positions, positions dropped at the front)], in memory and as dense arrays per sequence."""

    def __init__(self, dev, rng, seqs, kvH, hs, page, order, half, spare=2, width=None, pad=0, fill=True, missing=-1.0):
        self.dev, self.seqs, self.kvH, self.hs, self.page, self.order, self.half = dev, seqs, kvH, hs, page, order, half
        self.width = width or max(1, max(-(-m // page) for _, m, _ in seqs))
        need = sum(-(-m // page) for _, m, _ in seqs)
        self.pages = need + spare
        shape = (self.pages, kvH, page, hs)
        self.k, self.v = np.full(shape, np.nan, np.float32), np.full(shape, np.nan, np.float32)
        perm, at = rng.permutation(self.pages), 0
        self.table = np.full((len(seqs), self.width), missing, np.float32)
        self.dense = []
        for b, (n, m, gone) in enumerate(seqs):
            ids = perm[at:at + -(-m // page)]
            at += len(ids)
            self.table[b, :len(ids)] = ids
            self.table[b, :gone // page] = missing
            k, v = (rounded(rng.standard_normal((m, kvH, hs)), half) for _ in range(2))
            for t in range(gone if fill else m, m):
                self.k[ids[t // page], :, t % page], self.v[ids[t // page], :, t % page] = k[t], v[t]
            self.dense.append((k, v))
        new = [n for n, _, _ in seqs]
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.float32)
        self.tokens = int(sum(new)) + pad
        self.lens = np.float32([m for _, m, _ in seqs])
        self.h = dict(k=dev.put(self.laid(self.k), half), v=dev.put(self.laid(self.v), half), table=dev.put(self.table), starts=dev.put(self.starts), lens=dev.put(self.lens))

    def laid(self, a):
        return a if self.order == "head" else np.ascontiguousarray(a.transpose(0, 2, 1, 3))

    def get(self, name):
        shape = (self.pages, self.kvH, self.page, self.hs)
        a = self.dev.get(self.h[name])
        return a.reshape(shape) if self.order == "head" else a.reshape(self.pages, self.page, self.kvH, self.hs).transpose(0, 2, 1, 3)

    @property
    def strides(self):
        whole = self.kvH * self.page * self.hs
        return (whole, self.page * self.hs, self.hs) if self.order == "head" else (whole, self.hs, self.kvH * self.hs)

    def attend(self, q, y, H, **more):
        self.dev.cuda.AttnPagedForward(len(self.seqs), self.tokens, H, self.kvH, self.hs, self.pages, self.page, self.width, q, self.h["k"], self.h["v"],
                                       self.h["table"], self.h["starts"], self.h["lens"], y, *self.strides, **more)

    def append(self, qkv, q, H, **more):
        self.dev.cuda.PagedAppend(len(self.seqs), self.tokens, H, self.kvH, self.hs, self.pages, self.page, self.width, qkv, q, self.h["k"], self.h["v"],
                                  self.h["table"], self.h["starts"], self.h["lens"], *self.strides, **more)


def attention(c, q, H, weights16, scale=None, out16=False):
    """y and its tolerance, of every token; rows past the sequences are NaN in both."""
    G, hs = H // c.kvH, c.hs
    scale = hs ** -0.5 if scale is None else scale
    y, tol = np.full((c.tokens, H, hs), np.nan), np.full((c.tokens, H, hs), np.nan)
    at = 0
    for i, ((n, m, gone), (k, v)) in enumerate(zip(c.seqs, c.dense)):
        there = np.arange(m) >= gone
        for a, b in getattr(c, "holes", {}).get(i, ()):
            there[a:b] = False
        sees = there[None, :] & (np.arange(m)[None, :] <= np.arange(m - n, m)[:, None])
        some = sees.any(1)
        for h in range(H):
            # what nobody sees may be anything
            kk, vv = (np.where(there[:, None], x[:, h // G].astype(np.float64), 0) for x in (k, v))
            qq = q[at:at + n, h].astype(np.float64)
            s = np.where(sees, scale * (qq @ kk.T), -np.inf)
            s = s - np.where(some, s.max(1, initial=-np.inf), 0)[:, None]
            e = np.exp(s)
            w = e / np.where(some, e.sum(1), 1)[:, None]
            # scores: a dot product of hs terms, its scaling, the exponential's argument and the exponential
            size = abs(scale) * (abs(qq) @ abs(kk).T)
            ds = (hs + 8) * U32 * np.where(sees, size, 0).max(1, initial=0) + 4 * U32 * np.where(sees, abs(s), 0).max(1, initial=0) + 4 * U32
            # weights each off by 2 ds (theirs and their sum's), rounded to 16 bits where the products are; sums of all of them
            off = 2 * ds + (2 * U16 if weights16 else 0) + (sees.sum(1) + 8) * U32
            y[at:at + n, h] = w @ vv
            tol[at:at + n, h] = off[:, None] * (w @ abs(vv)) + (U16 if out16 else U32) * abs(y[at:at + n, h]) + 1e-30
            tol[at:at + n, h][~some] = 0
        at += n
    return y, tol


def check_attention(dev, rng, c, H, act16, scale=0.0, max_new=0):
    q = rounded(rng.standard_normal((c.tokens, H, c.hs)) * 1.5, act16)
    hq, hy = dev.put(q, act16), dev.put(np.full(q.size, 7.0, np.float32), act16)
    c.attend(hq, hy, H, fScale=scale, nMaxNew=max_new)
    got = dev.get(hy, q.shape)
    c.attend(hq, hy, H, fScale=scale, nMaxNew=max_new)
    assert np.array_equal(got, dev.get(hy, q.shape), equal_nan=True)      # the same bits every time
    want, tol = attention(c, q, H, act16, scale or None, act16)
    live = sum(n for n, _, _ in c.seqs)
    assert np.isfinite(got).all()
    worst = (abs(got[:live] - want[:live]) - tol[:live]).max() if live else -1
    assert worst <= 0, "off by %.3g more than the roundings" % worst
    assert (got[live:] == 7.0).all()          # rows behind the last sequence
    return got


TYPES = [(False, False), (False, True), (True, True)]      # 16-bit rows, 16-bit cache
SHAPES = [
    # name, H, kvH, hs, page, order, [(new, positions, dropped)], padding rows
    ("one", 2, 2, 64, 16, "head", [(1, 1, 0)], 0),
    ("one_page_inside", 4, 1, 64, 16, "pos", [(1, 37, 0)], 3),
    ("steps", 8, 2, 128, 16, "head", [(1, 5, 0), (1, 129, 0), (1, 64, 0), (1, 300, 0)], 0),
    ("groups_of_seven", 7, 1, 64, 8, "pos", [(1, 70, 0), (3, 9, 0)], 0),
    ("chunks", 4, 2, 64, 32, "head", [(40, 40, 0), (70, 200, 0), (1, 33, 0), (17, 90, 0)], 5),
    ("chunk_wide", 6, 2, 128, 16, "pos", [(150, 333, 0), (1, 128, 0)], 1),
    ("empty_ones", 4, 4, 32, 16, "head", [(0, 0, 0), (2, 50, 0), (0, 20, 0), (1, 1, 0), (0, 0, 0)], 2),
    ("more_new_than_positions", 2, 1, 64, 16, "head", [(20, 7, 0), (5, 2, 0)], 0),
    ("no_positions", 2, 2, 64, 16, "head", [(3, 0, 0), (2, 40, 0)], 0),
    ("dropped", 4, 2, 64, 16, "pos", [(5, 100, 64), (1, 48, 32), (30, 95, 16)], 0),
    ("all_dropped", 2, 1, 128, 8, "head", [(1, 32, 32), (4, 30, 24), (1, 200, 184)], 0),
    ("size_48", 6, 6, 48, 16, "head", [(1, 77, 0), (33, 60, 0)], 0),
    ("size_80", 4, 2, 80, 24, "pos", [(1, 150, 0), (20, 45, 0)], 0),
    ("size_6", 3, 3, 6, 5, "pos", [(1, 21, 0), (9, 12, 0)], 0),
    ("size_256", 2, 1, 256, 16, "head", [(1, 50, 0), (18, 40, 0)], 0),
    ("size_198", 2, 2, 198, 7, "pos", [(1, 50, 0), (3, 9, 0)], 0),
    ("long", 4, 2, 64, 64, "head", [(1, 5000, 0)], 0),
    ("many", 2, 1, 32, 8, "head", [(1 + b % 3, 3 + 7 * b % 61, 0) for b in range(200)], 0),
    ("more_than_a_scan", 1, 1, 32, 16, "pos", [(b % 3, (b % 3) + 11 * b % 40, 0) for b in range(600)], 1),
    ("heads_of_two_tiles", 20, 1, 64, 16, "head", [(1, 200, 0), (2, 30, 0), (40, 60, 0)], 0),
    ("more_tiles_than_workgroups_at_once", 8, 8, 64, 16, "head", [(65 + b % 3, 65 + b % 3 + 5 * b % 30, 0) for b in range(70)], 4),
    ("a_prompt", 4, 1, 128, 16, "pos", [(400, 400, 0), (90, 700, 48)], 0),
    ("long_and_short", 4, 1, 128, 32, "pos", [(1, 3000, 0), (1, 1, 0), (2, 700, 0), (0, 500, 0), (1, 64, 0)], 0),
]


@pytest.mark.parametrize("act16,cache16", TYPES)
@pytest.mark.parametrize("name,H,kvH,hs,page,order,seqs,pad", SHAPES, ids=[s[0] for s in SHAPES])
def test_attention(dev, name, H, kvH, hs, page, order, seqs, pad, act16, cache16):
    rng = np.random.default_rng(len(name) + hs)
    # "more_new_than_positions": token j stands at a negative position and sees nothing
    c = Cache(dev, rng, seqs, kvH, hs, page, order, cache16, pad=pad)
    check_attention(dev, rng, c, H, act16)


@pytest.mark.parametrize("act16,cache16", TYPES)
@pytest.mark.parametrize("missing", [-1.0, np.nan, np.inf, -np.inf, 1e9, 4294967296.0])
def test_entries_that_are_no_page(dev, act16, cache16, missing):
    rng = np.random.default_rng(5)
    c = Cache(dev, rng, [(1, 90, 48), (20, 70, 32), (2, 64, 64)], 2, 64, 16, "head", cache16, width=9, missing=missing)
    check_attention(dev, rng, c, 4, act16)


@pytest.mark.parametrize("act16,cache16", TYPES)
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_later_tokens_have_no_say(dev, act16, cache16, bad):
    """Infinities and NaN in the keys and values of a chunk's later tokens have no part in the rows before them.  (Those rows may be added up in
    another order then, so it is the definition that they are held to, with its tolerance, and not the bits of a call without them.)"""
    rng = np.random.default_rng(6)
    H, kvH, hs, n, m = 4, 2, 64, 50, 130
    q = rounded(rng.standard_normal((n, H, hs)), act16)
    out = []
    for at in (None, m - 20):
        c = Cache(dev, np.random.default_rng(7), [(n, m, 0)], kvH, hs, 16, "head", cache16)
        if at is not None:
            page, slot = int(c.table[0, at // 16]), at % 16
            for a in (c.k, c.v):
                a[page, :, slot, [3, 40]] = bad
            c.h["k"], c.h["v"] = dev.put(c.laid(c.k), cache16), dev.put(c.laid(c.v), cache16)
        hq, hy = dev.put(q, act16), dev.zeros(q.size, act16)
        c.attend(hq, hy, H)
        out.append(dev.get(hy, q.shape))
    want, tol = attention(Cache(dev, np.random.default_rng(7), [(n, m, 0)], kvH, hs, 16, "head", cache16), q, H, act16, None, act16)
    assert (abs(out[0] - want) <= tol).all()
    assert (abs(out[1] - want)[:n - 20] <= tol[:n - 20]).all()
    assert np.isnan(out[1][n - 20:]).any(axis=(1, 2)).all()


@pytest.mark.parametrize("act16,cache16", TYPES)
def test_scores_far_from_zero(dev, act16, cache16):
    """Rows whose weights lie at one position, at scores in the hundreds either way."""
    rng = np.random.default_rng(8)
    c = Cache(dev, rng, [(1, 200, 0), (40, 100, 0)], 2, 64, 16, "head", cache16)
    check_attention(dev, rng, c, 4, act16, scale=20.0)
    check_attention(dev, rng, c, 4, act16, scale=-20.0)
    check_attention(dev, rng, c, 4, act16, scale=1e-3)


@pytest.mark.parametrize("act16,cache16", TYPES)
def test_scores_that_are_all_minus_infinity(dev, act16, cache16):
    """no weights: NaN, as a softmax over them has it; the sequences beside it are not touched"""
    rng = np.random.default_rng(9)
    c = Cache(dev, rng, [(1, 40, 0), (3, 60, 0)], 1, 64, 16, "head", cache16)
    q = rounded(np.abs(rng.standard_normal((4, 1, 64))) + 1, act16)
    for t in range(40):
        c.k[int(c.table[0, t // 16]), :, t % 16] = -np.inf
    c.h["k"] = dev.put(c.laid(c.k), cache16)
    hq, hy = dev.put(q, act16), dev.zeros(q.size, act16)
    c.attend(hq, hy, 1)
    got = dev.get(hy, q.shape)
    assert np.isnan(got[0]).all() and np.isfinite(got[1:]).all()


@pytest.mark.parametrize("act16,cache16", TYPES)
@pytest.mark.parametrize("n", [1, 60])
def test_keys_of_infinity(dev, act16, cache16, n):
    """Scores of -inf are weights of zero and nothing else; a query that is no number spoils its own row alone."""
    rng = np.random.default_rng(15)
    H, kvH, hs, m = 2, 1, 64, 100
    q = rounded(abs(rng.standard_normal((n, H, hs))) + 0.1, act16)
    c = Cache(dev, rng, [(n, m, 0)], kvH, hs, 16, "head", cache16)
    k, v = c.dense[0]
    for at in (3, 35, 36):
        k[at] = -np.inf
        c.k[int(c.table[0, at // 16]), :, at % 16] = -np.inf
    c.h["k"] = dev.put(c.laid(c.k), cache16)
    q[n - 1, 1, 7] = np.nan
    hq, hy = dev.put(q, act16), dev.zeros(q.size, act16)
    c.attend(hq, hy, H)
    got = dev.get(hy, q.shape)
    assert np.isnan(got[n - 1, 1]).all()
    keep = [t for t in range(m) if t not in (3, 35, 36)]
    for j in range(n):
        for h in range(H - (j == n - 1)):
            seen = [t for t in keep if t <= m - n + j]
            s = k[seen, 0].astype(np.float64) @ q[j, h] / 8
            e = np.exp(s - s.max())
            w = e / e.sum()
            vv = v[seen, 0].astype(np.float64)
            # as attention() counts it
            off = 2 * ((hs + 8) * U32 * (abs(k[seen, 0].astype(np.float64)) @ abs(q[j, h])).max() / 8 + 4 * U32 * abs(s - s.max()).max() + 4 * U32) + (
                2 * U16 if act16 else 0) + (len(w) + 8) * U32
            assert (abs(got[j, h] - w @ vv) <= off * (w @ abs(vv)) + (U16 if act16 else U32) * abs(w @ vv)).all()


@pytest.mark.parametrize("act16,cache16", TYPES)
@pytest.mark.parametrize("size", [1e-30, 1e30, 3e38])
def test_values_far_from_one(dev, act16, cache16, size):
    """Values at the ends of the range come out as large as they went in."""
    rng = np.random.default_rng(16)
    H, kvH, hs, n, m = 1, 1, 64, 40, 90
    c = Cache(dev, rng, [(n, m, 0)], kvH, hs, 16, "head", cache16)
    k, v = c.dense[0]
    v[:] = rounded(size * np.sign(v) * (1 + 0.1 * rng.random(v.shape)), cache16)
    for t in range(m):
        c.v[int(c.table[0, t // 16]), :, t % 16] = v[t]
    c.h["v"] = dev.put(c.laid(c.v), cache16)
    q = np.float32(np.zeros((n, H, hs)))
    if size > 1e38:
        v_ = v.copy()       # a mean of numbers of one sign, so that no sum leaves the range before it is divided
        k[:] = 0
        for t in range(m):
            c.k[int(c.table[0, t // 16]), :, t % 16] = 0
            c.v[int(c.table[0, t // 16]), :, t % 16] = abs(v_[t]) / 512
        c.h["k"], c.h["v"] = dev.put(c.laid(c.k), cache16), dev.put(c.laid(c.v), cache16)
        v[:] = rounded(abs(v_) / 512, cache16)
    hq, hy = dev.put(q, act16), dev.zeros(q.size, act16)
    c.attend(hq, hy, H)
    got = dev.get(hy, q.shape)
    for j in range(n):
        vv = v[:m - n + j + 1, 0].astype(np.float64)
        tol = ((len(vv) + 12) * U32 + (2 * U16 if act16 else 0)) * abs(vv).mean(0) + (U16 if act16 else U32) * abs(vv.mean(0))
        assert (abs(got[j, 0] - vv.mean(0)) <= tol).all()


# Long chunks in 16-bit storage, enough tiles of 256 rows for the chip: heads and new tokens by the hundred
LONG = [
    # name, H, kvH, hs, page, order, [(new, positions, dropped)], padding rows
    ("prompt", 128, 128, 64, 16, "head", [(300, 300, 0)], 3),
    ("chunk_of_four_heads", 512, 128, 64, 32, "pos", [(70, 401, 0)], 0),
    ("wide_two_sequences", 128, 64, 128, 16, "head", [(260, 517, 0), (140, 140, 0)], 0),
    ("groups_of_seven", 448, 64, 128, 8, "pos", [(80, 300, 0), (37, 40, 0)], 1),
    ("dropped", 128, 128, 64, 24, "head", [(270, 700, 168)], 0),
    ("dropped_into_the_chunk", 128, 128, 64, 16, "head", [(300, 400, 160)], 0),
    ("single_tokens_beside", 256, 64, 128, 16, "head", [(200, 500, 0), (1, 900, 0), (3, 70, 0), (0, 5, 0), (150, 160, 0)], 2),
    ("more_new_than_positions", 128, 128, 64, 16, "head", [(300, 270, 0)], 0),
    ("a_page_to_a_tile", 128, 64, 128, 128, "pos", [(320, 1000, 0)], 0),
]


@pytest.mark.parametrize("scale", [0.0, -0.2, 6.0])
@pytest.mark.parametrize("name,H,kvH,hs,page,order,seqs,pad", LONG, ids=[s[0] for s in LONG])
def test_long_chunks(dev, name, H, kvH, hs, page, order, seqs, pad, scale):
    rng = np.random.default_rng(hs + len(name))
    check_attention(dev, rng, Cache(dev, rng, seqs, kvH, hs, page, order, True, pad=pad), H, True, scale=scale)


@pytest.mark.parametrize("act16,cache16", TYPES)
def test_holes(dev, act16, cache16):
    """Pages given up in the middle of sequences: the first page and a window kept, say."""
    for H, kvH, hs, seqs in ((128, 128, 64, [(300, 700, 0)]), (4, 2, 64, [(40, 200, 0), (1, 300, 0), (2, 130, 0)])):
        rng = np.random.default_rng(17)
        c = Cache(dev, rng, seqs, kvH, hs, 16, "head", cache16)
        c.holes = {}
        for b, (n, m, _) in enumerate(seqs):
            c.holes[b] = [(16, 16 * ((m - n) // 32))]
            c.table[b, 1:(m - n) // 32] = -1
        c.h["table"] = dev.put(c.table)
        check_attention(dev, rng, c, H, act16)


@pytest.mark.parametrize("bad", [np.inf, np.nan])
@pytest.mark.parametrize("where", ["k", "v", "q"])
def test_long_chunks_with_values_that_are_not_finite(dev, where, bad):
    rng = np.random.default_rng(18)
    H, kvH, hs, n, m, at = 128, 128, 64, 280, 340, 250
    c = Cache(dev, rng, [(n, m, 0)], kvH, hs, 16, "head", True)
    q = rounded(rng.standard_normal((n, H, hs)), True)
    want, tol = attention(c, q, H, True, None, True)
    if where == "q":
        q[at, :, 5] = bad
        rows, touched = np.arange(n) != at, np.arange(n) == at
    else:
        a = c.k if where == "k" else c.v
        a[int(c.table[0, (m - n + at) // 16]), :, (m - n + at) % 16, 5] = bad
        c.h[where] = dev.put(c.laid(a), True)
        rows = np.arange(n) < at
        touched = ~rows
    hq, hy = dev.put(q, True), dev.zeros(q.size, True)
    c.attend(hq, hy, H)
    got = dev.get(hy, q.shape)
    assert (abs(got - want)[rows] <= tol[rows]).all()
    if where != "k":      # (a key's infinity may be a weight of zero)
        assert not np.isfinite(got[touched]).all(axis=2).any()


@pytest.mark.parametrize("act16,cache16", TYPES)
@pytest.mark.parametrize("max_new", [1, 40, 500])
def test_hint(dev, act16, cache16, max_new):
    """The bound on new tokens changes nothing but kernels, even where it does not hold."""
    rng = np.random.default_rng(10)
    c = Cache(dev, rng, [(40, 90, 0), (1, 70, 0), (33, 33, 0)], 2, 64, 16, "pos", cache16)
    check_attention(dev, rng, c, 4, act16, max_new=max_new)


def test_odd_strides_and_addresses(dev):
    """A cache at an odd element, rows of other lengths, keys and values of a position side by side."""
    rng = np.random.default_rng(11)
    for half in (False, True):
        for lead in (0, 1, 8):
            kvH, hs, page, seqs = 2, 64, 16, [(1, 50, 0), (9, 40, 0)]
            c = Cache(dev, rng, seqs, kvH, hs, page, "head", half)
            sT = 2 * hs + lead
            sH, sP = page * sT + lead, kvH * (page * sT + lead) + 5 * lead
            mem = np.full(lead + c.pages * sP + hs, np.nan, np.float32)
            for a, off in ((c.k, lead), (c.v, lead + hs)):
                for p in range(c.pages):
                    for h in range(kvH):
                        for t in range(page):
                            at = off + p * sP + h * sH + t * sT
                            mem[at:at + hs] = a[p, h, t]
            base = dev.put(mem, half)
            n = mem.size - lead - hs
            c.h["k"] = dev.cuda.CreateMemoryPointer(base, lead, n)
            c.h["v"] = dev.cuda.CreateMemoryPointer(base, lead + hs, n)
            Cache.strides, keep = property(lambda self: (sP, sH, sT)), Cache.strides
            try:
                check_attention(dev, rng, c, 4, half)
                # and new tokens into it
                qkv = rounded(rng.standard_normal((c.tokens, 8 * hs)), half)
                hq = dev.zeros(c.tokens * 4 * hs, half)
                c.append(dev.put(qkv, half), hq, 4)
            finally:
                Cache.strides = keep
            after = dev.get(base)
            rows = qkv.reshape(c.tokens, 8, hs)
            i = 0
            for b, (new, m, _) in enumerate(seqs):
                for t in range(m - new, m):
                    for h in range(kvH):
                        at = lead + int(c.table[b, t // page]) * sP + h * sH + (t % page) * sT
                        mem[at:at + hs], mem[at + hs:at + 2 * hs] = rows[i, 4 + h], rows[i, 6 + h]
                    i += 1
            assert np.array_equal(after, mem, equal_nan=True)
            dev.cuda.FreeMemoryPointer(c.h["k"])
            dev.cuda.FreeMemoryPointer(c.h["v"])


def test_cache_past_32_bits(dev):
    """Pages more than 2^32 values from the first."""
    rng = np.random.default_rng(12)
    H, kvH, hs, page, far = 2, 1, 64, 16, (1 << 31) + 64
    cuda = dev.cuda
    hk, hv = cuda.AllocMemory(2 * far + page * hs, bHalfSize=True), cuda.AllocMemory(2 * far + page * hs, bHalfSize=True)
    try:
        k, v = (rounded(rng.standard_normal((20, kvH, hs)), True) for _ in range(2))
        table, starts, lens = dev.put(np.float32([[2, 1]])), dev.put(np.float32([0, 2])), dev.put(np.float32([20]))
        rows = np.concatenate([rounded(rng.standard_normal((20, H * hs)), True), k.reshape(20, -1), v.reshape(20, -1)], 1)
        # the whole sequence in through the append, then attention of its last two tokens
        all_starts = dev.put(np.float32([0, 20]))
        q20 = dev.zeros(20 * H * hs, True)
        cuda.PagedAppend(1, 20, H, kvH, hs, 3, page, 2, dev.put(rows, True), q20, hk, hv, table, all_starts, lens, far, page * hs, hs)
        q = rows[18:, :H * hs].reshape(2, H, hs)
        hq, hy = dev.put(q, True), dev.zeros(q.size, True)
        cuda.AttnPagedForward(1, 2, H, kvH, hs, 3, page, 2, hq, hk, hv, table, starts, lens, hy, far, page * hs, hs)
        c = type("C", (), dict(kvH=kvH, hs=hs, tokens=2, seqs=[(2, 20, 0)], dense=[(k, v)]))
        want, tol = attention(c, q, H, True, None, True)
        assert (abs(dev.get(hy, q.shape) - want) <= tol).all()
    finally:
        cuda.FreeMemory(hk)
        cuda.FreeMemory(hv)


# ---- new tokens into the pages ---------------------------------------------------------------------------------------------------
def turned(x, pos):
    """x (tokens, heads, hs) turned to its position"""
    hs = x.shape[-1]
    a = np.asarray(pos, np.float64)[:, None, None] * THETA ** (-np.arange(0, hs, 2) / hs)
    z = (x[..., 0::2] + 1j * x[..., 1::2]) * np.exp(1j * a)
    return np.stack([z.real, z.imag], -1).reshape(x.shape)


def head_norm(x, w):
    x = x.astype(np.float64)
    return w * x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS)


def pair_size(x):
    """magnitude of every value's pair: what a rotation's roundings are relative to"""
    s = np.hypot(x[..., 0::2], x[..., 1::2])
    return np.repeat(s, 2, -1)


APPENDS = [
    ("one", 2, 2, 64, 16, "head", [(1, 1, 0)], 0),
    ("steps", 8, 2, 128, 16, "pos", [(1, 5, 0), (1, 129, 0), (1, 64, 0)], 2),
    ("chunks", 12, 4, 64, 32, "head", [(40, 40, 0), (70, 200, 0), (0, 9, 0), (17, 90, 0)], 5),
    ("size_48", 6, 6, 48, 16, "pos", [(1, 77, 0), (33, 60, 0)], 0),
    ("size_6", 3, 3, 6, 5, "head", [(1, 21, 0), (9, 12, 0)], 1),
    ("size_256", 2, 1, 256, 8, "pos", [(3, 50, 0)], 0),
    ("size_198", 2, 1, 198, 8, "pos", [(3, 50, 0)], 0),
    ("before_zero", 2, 1, 64, 16, "head", [(5, 3, 0), (2, 0, 0), (1, 4, 0)], 0),
    ("not_given", 2, 1, 64, 16, "head", [(5, 32, 32), (3, 40, 0)], 0),
    ("many", 2, 1, 32, 8, "head", [(b % 4, 3 + b % 4 + 7 * b % 61, 0) for b in range(150)], 3),
    ("wide_row", 40, 40, 64, 16, "pos", [(700, 900, 0)], 0),
]


@pytest.mark.parametrize("act16,cache16", TYPES)
@pytest.mark.parametrize("norm,rope", [(False, False), (False, True), (True, False), (True, True)])
@pytest.mark.parametrize("name,H,kvH,hs,page,order,seqs,pad", APPENDS, ids=[s[0] for s in APPENDS])
def test_append(dev, name, H, kvH, hs, page, order, seqs, pad, norm, rope, act16, cache16):
    rng = np.random.default_rng(hs + H)
    c = Cache(dev, rng, seqs, kvH, hs, page, order, cache16, pad=pad, fill=False)
    before = dict(k=c.k.copy(), v=c.v.copy())
    x = rounded(rng.standard_normal((c.tokens, H + 2 * kvH, hs)) * 2, act16)
    w = [rounded(1 + 0.2 * rng.standard_normal(hs), act16) for _ in range(2)]
    hq = dev.put(np.full((c.tokens, H, hs), 7.0, np.float32), act16)
    hr = dev.cuda.CreateRope(0, 0, 1, 1, c.width * page, H, hs, THETA) if rope else 0
    c.append(dev.put(x, act16), hq, H, hRope=hr, bNorm=norm, hWq=dev.put(w[0], act16) if norm else 0, hWk=dev.put(w[1], act16) if norm else 0, fEps=EPS)
    pos = np.concatenate([np.arange(m - n, m) for n, m, _ in seqs]) if c.tokens > pad else np.zeros(0, int)
    live = len(pos)
    q, k, v = (t.astype(np.float64) for t in np.split(x[:live], [H, H + kvH], 1))
    if norm:
        q, k = head_norm(q, w[0].astype(np.float64)), head_norm(k, w[1].astype(np.float64))
    size = dict(q=pair_size(q) if rope else abs(q), k=pair_size(k) if rope else abs(k), v=abs(v))
    if rope:
        q, k = turned(q, np.maximum(pos, 0)), turned(k, np.maximum(pos, 0))
    # the mean of squares: hs roundings of its terms, halved by the root; root, quotient, two products; two products and their sum with a rounded cosine and sine
    off = ((hs + 2) * U32 / 2 + 6 * U32 if norm else 0) + (4 * U32 if rope else 0)
    tol = lambda n, want, half: off * size[n] + (U16 if half else U32) * abs(want) + 1e-37  # noqa: E731
    got = dev.get(hq, (c.tokens, H, hs))
    assert (abs(got[:live] - q) <= tol("q", q, act16)).all()
    assert (got[live:] == 7.0).all()
    for name_, want in (("k", k), ("v", v)):
        pages, i = c.get(name_), 0
        expect = before[name_]
        for b, (n, m, gone) in enumerate(seqs):
            for p in range(m - n, m):
                at = c.table[b, p // page] if p >= 0 else -1
                if at >= 0:
                    g = pages[int(at), :, p % page]
                    t = tol(name_, want, cache16)[i] if name_ == "k" else (U16 if cache16 and not act16 else 0) * abs(want[i])
                    assert (abs(g - want[i]) <= t).all()
                    expect[int(at), :, p % page] = g
                i += 1
        assert np.array_equal(pages, expect, equal_nan=True)      # nothing else has been written
    if hr:
        dev.cuda.FreeRope(hr)


def test_far_positions_turn_by_their_angle(dev):
    """Position 65000 at fp32 precision: an angle in fp32 would be off by 65000 u."""
    rng = np.random.default_rng(13)
    H, kvH, hs, page, m = 1, 1, 64, 64, 65000
    hr = dev.cuda.CreateRope(0, 0, 1, 1, 1016 * page, H, hs, THETA)
    x = np.float32(rng.standard_normal((1, 3, hs)))
    table = np.full((1, 1016), -1, np.float32)
    table[0, (m - 1) // page] = 0
    hq, hk, hv = dev.zeros(hs), dev.zeros(page * hs), dev.zeros(page * hs)
    dev.cuda.PagedAppend(1, 1, H, kvH, hs, 1, page, 1016, dev.put(x), hq, hk, hv, dev.put(table), dev.put(np.float32([0, 1])), dev.put(np.float32([m])),
                         page * hs, page * hs, hs, hr)
    got = dev.get(hk, (page, hs))[(m - 1) % page]
    want = turned(x[:, 1:2].astype(np.float64), [m - 1])[0, 0]
    assert (abs(got - want) <= 5 * U32 * pair_size(want[None])[0]).all()
    dev.cuda.FreeRope(hr)


# ---- the two together, as a server runs them ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("act16,cache16", TYPES)
def test_prompts_in_chunks_and_steps(dev, act16, cache16):
    """Three sequences come in over nine calls, in chunks and single tokens, pages handed out as they grow; every call's attention is that of the
    whole sequence so far."""
    rng = np.random.default_rng(14)
    H, kvH, hs, page, width = 4, 2, 64, 16, 8
    totals = [100, 37, 61]
    plans = [[40, 0, 3], [40, 30, 1], [0, 1, 1], [17, 1, 50], [1, 1, 1], [1, 1, 1], [1, 1, 1], [0, 1, 2], [0, 1, 1]]
    assert [sum(p[b] for p in plans) for b in range(3)] == totals
    rows = [rounded(rng.standard_normal((t, H + 2 * kvH, hs)), act16) for t in totals]
    pages = list(rng.permutation(24))
    table = np.full((3, width), -1, np.float32)
    hk, hv, hr = dev.put(np.full(24 * kvH * page * hs, np.nan, np.float32), cache16), dev.put(np.full(24 * kvH * page * hs, np.nan, np.float32), cache16), 0
    hr = dev.cuda.CreateRope(0, 0, 1, 1, width * page, H, hs, THETA)
    have = [0, 0, 0]
    w = [rounded(1 + 0.2 * rng.standard_normal(hs), act16) for _ in range(2)]
    hw = [dev.put(x, act16) for x in w]
    strides = (kvH * page * hs, page * hs, hs)
    for plan in plans:
        new = np.concatenate([rows[b][have[b]:have[b] + n] for b, n in enumerate(plan)])
        have = [a + n for a, n in zip(have, plan)]
        for b in range(3):
            for e in range(-(-have[b] // page)):
                if table[b, e] < 0:
                    table[b, e] = pages.pop()
        ht, hs_, hl = dev.put(table), dev.put(np.float32(np.concatenate([[0], np.cumsum(plan)]))), dev.put(np.float32(have))
        N = len(new)
        hq, hy = dev.zeros(N * H * hs, act16), dev.zeros(N * H * hs, act16)
        dev.cuda.PagedAppend(3, N, H, kvH, hs, 24, page, width, dev.put(new, act16), hq, hk, hv, ht, hs_, hl, *strides, hr, True, *hw, EPS)
        dev.cuda.AttnPagedForward(3, N, H, kvH, hs, 24, page, width, hq, hk, hv, ht, hs_, hl, hy, *strides)
        got, q = dev.get(hy, (N, H, hs)), dev.get(hq, (N, H, hs))
        dense = []
        for b in range(3):
            x = rows[b][:have[b]].astype(np.float64)
            dense.append((rounded(turned(head_norm(x[:, H:H + kvH], w[1].astype(np.float64)), np.arange(have[b])), cache16), rounded(x[:, H + kvH:], cache16)))
        c = type("C", (), dict(kvH=kvH, hs=hs, tokens=N, seqs=[(n, m, 0) for n, m in zip(plan, have)], dense=dense))
        want, tol = attention(c, q, H, act16, None, act16)
        # keys that the call rounded the other way than the 64-bit norm: one step of their type, which the scores' tolerance takes hs times over
        slack = (2 * U16 if cache16 else 64 * U32) * 2 * np.sqrt(hs) * np.abs(q).max() * 4 / np.sqrt(hs)
        assert (abs(got - want) <= tol + slack).all()
    dev.cuda.FreeRope(hr)


# ---- refusals ---------------------------------------------------------------------------------------------------------------------
def refused(code, f, *a, **k):
    with pytest.raises(CudaDnnError) as e:
        f(*a, **k)
    assert e.value.code == code, e.value


def test_attention_refusals(dev):
    B, N, H, kvH, hs, pages, page, width = 2, 3, 4, 2, 64, 5, 16, 2
    q, y = dev.zeros(N * H * hs), dev.zeros(N * H * hs)
    n = pages * kvH * page * hs
    k, v, k16 = dev.zeros(n), dev.zeros(n), dev.zeros(n, True)
    table, starts, lens = dev.zeros(B * width), dev.zeros(B + 1), dev.zeros(B)
    good = [B, N, H, kvH, hs, pages, page, width, q, k, v, table, starts, lens, y, kvH * page * hs, page * hs, hs]
    f = dev.cuda.AttnPagedForward
    f(*good)

    def bad(code, **change):
        names = "B N H kvH hs pages page width q k v table starts lens y sP sH sT".split()
        a = list(good)
        for name, value in change.items():
            a[names.index(name)] = value
        refused(code, f, *a)
    for name in ("B", "N", "H", "kvH", "hs", "pages", "page", "width"):
        bad(90001, **{name: 0})
        bad(90001, **{name: -1})
        bad(90001, **{name: 1 << 40})
    bad(90001, kvH=3)
    bad(90001, hs=63)
    bad(90001, hs=258)
    bad(90001, page=1 << 20, width=1 << 10)
    bad(90001, sT=-1)
    for name in ("q", "k", "v", "table", "starts", "lens", "y"):
        for h in (0, 9999):
            with pytest.raises(CudaDnnError):
                a = list(good)
                a["B N H kvH hs pages page width q k v table starts lens y sP sH sT".split().index(name)] = h
                f(*a)
    bad(90010, N=4)
    bad(90010, B=3)
    bad(90010, width=3)
    bad(90010, pages=6)
    bad(90010, sP=kvH * page * hs + 1)
    bad(90010, sT=1 << 62)
    bad(90011, k=k16)
    bad(90011, q=dev.zeros(N * H * hs, True))
    bad(90012, table=dev.zeros(B * width, True))
    bad(90012, lens=dev.zeros(B, True))
    for name in ("q", "k", "v"):
        bad(90001, y=good["B N H kvH hs pages page width q k v".split().index(name)])
    refused(90001, f, *good, nMaxNew=-1)
    # 16-bit rows over an fp32 cache
    refused(90011, f, *[dev.zeros(N * H * hs, True) if i in (8, 14) else x for i, x in enumerate(good)])


def test_append_refusals(dev):
    B, N, H, kvH, hs, pages, page, width = 2, 3, 4, 2, 64, 5, 16, 2
    qkv, q = dev.zeros(N * (H + 2 * kvH) * hs), dev.zeros(N * H * hs)
    n = pages * kvH * page * hs
    k, v, w = dev.zeros(n), dev.zeros(n), dev.zeros(hs)
    table, starts, lens = dev.zeros(B * width), dev.zeros(B + 1), dev.zeros(B)
    rope, short, other = (dev.cuda.CreateRope(0, 0, 1, 1, s, H, d, THETA) for s, d in ((width * page, hs), (width * page - 1, hs), (width * page, hs - 2)))
    good = [B, N, H, kvH, hs, pages, page, width, qkv, q, k, v, table, starts, lens, kvH * page * hs, page * hs, hs]
    names = "B N H kvH hs pages page width qkv q k v table starts lens sP sH sT".split()
    f = dev.cuda.PagedAppend
    f(*good, rope, True, w, w)

    def bad(code, *more, **change):
        a = list(good)
        for name, value in change.items():
            a[names.index(name)] = value
        refused(code, f, *a, *more)
    for name in names[:8]:
        bad(90001, **{name: 0})
    bad(90010, N=4)
    bad(90010, pages=6)
    bad(90001, sT=hs - 1)              # positions over one another
    bad(90001, sH=page * hs - 1)
    bad(90001, sP=kvH * page * hs - 1)
    bad(90001, sP=0)
    bad(90001, v=k)
    view = dev.cuda.CreateMemoryPointer(k, hs // 2, n - hs // 2)
    bad(90001, v=view, pages=4)
    dev.cuda.FreeMemoryPointer(view)
    bad(90001, q=qkv)
    bad(90001, k=qkv, pages=1, page=1)
    bad(90001, short)
    bad(90001, other)
    bad(90201, 77)
    bad(90011, rope, True, dev.zeros(hs, True), w)
    bad(90010, rope, True, dev.zeros(hs - 1), w)
    bad(90011, q=dev.zeros(N * H * hs, True))
    bad(90012, starts=dev.zeros(B + 1, True))
    refused(90001, f, *good, rope, True, w, w, float("nan"))
    refused(90001, f, *good, rope, True, w, w, -1.0)
    for r in (rope, short, other):
        dev.cuda.FreeRope(r)
