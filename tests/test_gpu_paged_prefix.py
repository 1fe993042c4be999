"""ATTN_PAGED_PREFIX_FWD (csrc/attn_prefix.hip) against the definition in 64 bits: attention of every sequence over its own pages, of which groups of sequences share the
first ones.  Caches, the definition and its tolerances are those of attention over pages; weights of 16-bit rows are counted as rounded to 16 bits, as there."""
import numpy as np
import pytest

from tests.conftest import Dev
from tests.test_gpu_paged import TYPES, U16, U32, Cache, attention, refused, rounded

pytestmark = pytest.mark.gpu


class Shared(Cache):
    """Sequences of which groups [(first, end, shared positions)] have their first positions in common: whole pages of them are the first sequence's, the rest of the
    positions has the same keys and values."""

    def __init__(self, dev, rng, seqs, groups, kvH, hs, page, order, half, wide=True, **more):
        # sequences that cannot hold this many bytes are not worth sharing for, and go to attention over pages: room for more than they have
        if wide:
            more["width"] = max(max(-(-m // page) for _, m, _ in seqs) + 1, int(125e6 / (len(seqs) * page * kvH * hs * (4 if half else 8))) + 1)
        super().__init__(dev, rng, seqs, kvH, hs, page, order, half, **more)
        self.groups = groups
        for first, end, shared in groups:
            for b in range(first + 1, end):
                n = min(shared, self.seqs[b][1], self.seqs[first][1])
                for p in range(-(-n // self.page)):
                    if (p + 1) * self.page <= n:
                        if self.table[b, p] >= 0:
                            self.k[int(self.table[b, p])] = self.v[int(self.table[b, p])] = np.nan
                        self.table[b, p] = self.table[first, p]
                for d, a in zip(self.dense[b], (self.k, self.v)):
                    d[:n] = self.dense[first][0 if a is self.k else 1][:n]
                    for t in range(n // self.page * self.page, n):
                        a[int(self.table[b, t // self.page]), :, t % self.page] = d[t]
        self.upload()

    def upload(self):
        dev = self.dev
        self.h.update(k=dev.put(self.laid(self.k), self.half), v=dev.put(self.laid(self.v), self.half), table=dev.put(self.table))
        if self.groups:
            self.h.update(groups=dev.put(np.float32([g[0] for g in self.groups] + [self.groups[-1][1]])), shared=dev.put(np.float32([g[2] for g in self.groups])))

    def attend_shared(self, q, y, H, **more):
        self.dev.cuda.AttnPagedPrefixForward(len(self.seqs), self.tokens, H, self.kvH, self.hs, self.pages, self.page, self.width, q, self.h["k"], self.h["v"],
                                             self.h["table"], self.h["starts"], self.h["lens"], y, *self.strides, len(self.groups), self.h["groups"], self.h["shared"], **more)


def check(dev, rng, c, H, act16, scale=0.0, max_new=0, q=None):
    q = rounded(rng.standard_normal((c.tokens, H, c.hs)) * 1.5, act16) if q is None else q
    hq, hy = dev.put(q, act16), dev.put(np.full(q.size, 7.0, np.float32), act16)
    c.attend_shared(hq, hy, H, fScale=scale, nMaxNew=max_new)
    got = dev.get(hy, q.shape)
    c.attend_shared(hq, hy, H, fScale=scale, nMaxNew=max_new)
    assert np.array_equal(got, dev.get(hy, q.shape), equal_nan=True)      # the same bits every time
    want, tol = attention(c, q, H, act16, scale or None, act16)
    live = sum(n for n, _, _ in c.seqs)
    assert np.isfinite(got).all()
    worst = (abs(got[:live] - want[:live]) - tol[:live]).max() if live else -1
    assert worst <= 0, "off by %.3g more than the roundings" % worst
    assert (got[live:] == 7.0).all()          # rows behind the last sequence
    return got


CASES = [
    # name, H, kvH, hs, page, order, [(new, positions, dropped)], [(first, end, shared)], padding rows
    ("two_tokens", 2, 2, 64, 16, "head", [(1, 33, 0), (1, 40, 0)], [(0, 2, 32)], 0),
    ("all_but_the_token", 4, 1, 64, 16, "pos", [(1, 33, 0)] * 5, [(0, 5, 32)], 1),
    ("one_sequence", 4, 2, 64, 16, "head", [(1, 100, 0)], [(0, 1, 64)], 0),
    ("nothing_shared", 4, 2, 64, 16, "head", [(1, 100, 0), (2, 30, 0)], [(0, 2, 0)], 0),
    ("less_than_a_page", 4, 2, 64, 16, "head", [(1, 100, 0), (2, 30, 0)], [(0, 2, 15)], 0),
    ("not_whole_pages", 8, 2, 128, 16, "head", [(1, 150, 0), (1, 141, 0), (1, 300, 0)], [(0, 3, 140)], 0),
    ("two_groups_and_others", 6, 3, 64, 8, "pos", [(1, 90, 0), (1, 70, 0), (1, 20, 0), (2, 200, 0), (1, 150, 0), (1, 44, 0), (1, 9, 0)], [(1, 3, 16), (3, 6, 40)], 2),
    ("groups_of_one", 4, 4, 64, 16, "head", [(1, 90, 0), (2, 170, 0), (1, 20, 0)], [(0, 1, 80), (1, 2, 160), (2, 3, 0)], 0),
    ("an_empty_group", 4, 4, 64, 16, "head", [(1, 90, 0), (2, 170, 0)], [(0, 0, 80), (0, 2, 64)], 0),
    ("chunks", 4, 2, 64, 32, "head", [(40, 140, 0), (70, 300, 0), (1, 133, 0), (17, 190, 0)], [(0, 4, 96)], 5),
    ("chunks_into_the_prefix", 4, 2, 64, 16, "head", [(60, 100, 0), (30, 200, 0), (1, 99, 0)], [(0, 3, 90)], 0),
    ("a_prompt_that_makes_the_prefix", 4, 2, 64, 16, "pos", [(64, 64, 0), (0, 64, 0), (0, 70, 0)], [(0, 3, 64)], 0),
    ("sequences_without_tokens", 4, 1, 64, 16, "head", [(0, 70, 0), (1, 90, 0), (0, 10, 0), (3, 80, 0), (0, 0, 0)], [(0, 5, 64)], 0),
    ("dropped_in_front", 4, 2, 64, 16, "pos", [(1, 100, 32), (5, 120, 32), (30, 195, 32)], [(0, 3, 64)], 0),
    ("all_of_it_dropped", 4, 2, 128, 16, "pos", [(1, 100, 64), (5, 120, 64), (1, 64, 64)], [(0, 3, 63)], 0),
    ("wide_chunks", 8, 2, 128, 16, "head", [(150, 400, 0), (90, 333, 0), (1, 250, 0)], [(0, 3, 200)], 3),
    ("groups_of_seven", 7, 1, 64, 8, "pos", [(1, 470, 0), (3, 409, 0), (1, 401, 0), (2, 500, 0)], [(0, 4, 400)], 0),
    ("heads_of_two_tiles", 40, 1, 64, 16, "head", [(1, 200, 0), (2, 130, 0), (20, 160, 0)], [(0, 3, 100)], 0),
    ("more_heads_than_a_chunk_tile", 160, 1, 64, 16, "head", [(1, 200, 0), (2, 130, 0)], [(0, 2, 100)], 0),
    ("size_48", 6, 6, 48, 16, "head", [(1, 177, 0), (33, 160, 0), (1, 99, 0)], [(0, 3, 96)], 0),
    ("size_80", 4, 2, 80, 24, "pos", [(1, 150, 0), (20, 145, 0)], [(0, 2, 100)], 0),
    ("size_6", 3, 3, 6, 5, "pos", [(1, 21, 0), (9, 22, 0)], [(0, 2, 12)], 0),
    ("size_256", 2, 1, 256, 16, "head", [(1, 150, 0), (18, 140, 0)], [(0, 2, 100)], 0),
    ("size_198", 2, 2, 198, 7, "pos", [(1, 50, 0), (3, 39, 0)], [(0, 2, 30)], 0),
    ("long", 4, 2, 64, 64, "head", [(1, 5000, 0), (1, 4500, 0), (1, 4481, 0)], [(0, 3, 4480)], 0),
    ("long_and_many", 4, 1, 128, 16, "pos", [(1, 3000 + 17 * b, 0) for b in range(40)], [(0, 40, 2990)], 0),
    ("many", 2, 1, 32, 8, "head", [(1 + b % 3, 53 + 7 * b % 61, 0) for b in range(200)], [(0, 90, 48), (90, 91, 48), (91, 200, 40)], 0),
    ("more_than_a_scan", 1, 1, 32, 16, "pos", [(b % 3, 40 + 11 * b % 40, 0) for b in range(600)], [(5, 400, 32), (400, 590, 16)], 1),
    ("as_many_groups_as_sequences", 2, 1, 64, 16, "head", [(1 + b % 2, 40 + b, 0) for b in range(300)], [(b, b + 1, 32) for b in range(300)], 0),
    ("single_tokens_of_unshared_heads", 4, 4, 64, 16, "head", [(1, 3000 + 17 * b, 0) for b in range(24)], [(0, 20, 2990), (20, 24, 100)], 0),
    ("unshared_heads_and_one_chunk", 3, 3, 48, 8, "pos", [(20, 900, 0)] + [(b % 2, 300 + b, 0) for b in range(40)], [(0, 30, 288), (30, 41, 64)], 2),
    ("more_groups_than_the_list_has", 1, 1, 32, 16, "head", [(1, 20 + b % 50, 0) for b in range(1100)], [(b, b + 1, 16) for b in range(1100)], 0),
    ("more_entries_than_the_list_has", 1, 1, 32, 16, "pos", [(1, 20 + b % 30, 0) for b in range(4090)], [(b * 409, b * 409 + 409, 16) for b in range(10)], 0),
    ("a_chunk_among_single_tokens", 4, 2, 64, 16, "head", [(150, 400, 0)] + [(1 + b % 3, 230 + 9 * b, 0) for b in range(24)], [(0, 25, 224)], 3),
    ("chunks_among_single_tokens", 8, 2, 128, 32, "pos", [(1, 400 + 5 * b, 0) if b % 6 else (60 + b, 500 + b, 0) for b in range(26)], [(0, 13, 384), (13, 26, 320)], 0),
    ("long_chunks_of_two_groups", 4, 4, 64, 16, "head", [(1, 1500 + 3 * b, 0) if b % 20 else (300 + b, 2000, 0) for b in range(60)], [(0, 30, 1400), (30, 60, 1024)], 1),
    ("three_groups_of_chunks", 8, 8, 64, 16, "head", [(65 + b % 3, 165 + b % 3 + 5 * b % 30, 0) for b in range(30)], [(0, 10, 96), (10, 11, 64), (11, 30, 80)], 4),
]


@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("act16,cache16", TYPES)
@pytest.mark.parametrize("name,H,kvH,hs,page,order,seqs,groups,pad", CASES, ids=[s[0] for s in CASES])
def test_against_the_definition(dev, name, H, kvH, hs, page, order, seqs, groups, pad, act16, cache16, wide):
    rng = np.random.default_rng(len(name) + hs)
    check(dev, rng, Shared(dev, rng, seqs, groups, kvH, hs, page, order, cache16, wide, pad=pad), H, act16)


@pytest.mark.parametrize("act16,cache16", TYPES)
@pytest.mark.parametrize("scale", [20.0, -20.0, 1e-3])
def test_scores_far_from_zero(dev, act16, cache16, scale):
    """Rows whose weights lie at one position, in the prefix or behind it."""
    rng = np.random.default_rng(8)
    c = Shared(dev, rng, [(1, 200, 0), (40, 190, 0), (3, 150, 0)], [(0, 3, 128)], 2, 64, 16, "head", cache16)
    check(dev, rng, c, 4, act16, scale=scale)


@pytest.mark.parametrize("act16,cache16", TYPES)
def test_holes_and_entries_that_are_no_page(dev, act16, cache16):
    for missing in (-1.0, np.nan, np.inf, 1e9):
        rng = np.random.default_rng(17)
        seqs = [(2, 200, 0), (40, 300, 0), (1, 130, 0)]
        c = Shared(dev, rng, seqs, [(0, 3, 96)], 2, 64, 16, "head", cache16, missing=missing)
        c.holes = {b: [(16, 64)] for b in range(3)}
        c.table[:, 1:4] = missing
        c.upload()
        check(dev, rng, c, 4, act16)


@pytest.mark.parametrize("act16,cache16", TYPES)
@pytest.mark.parametrize("wide", [True, False])
def test_first_sequences_of_groups_that_have_ended(dev, act16, cache16, wide):
    """Their rows of the block table name no pages any more, and count for nothing."""
    rng = np.random.default_rng(23)
    c = Shared(dev, rng, [(0, 150, 0), (0, 120, 0), (1, 140, 0), (2, 130, 0), (0, 99, 0), (1, 90, 0), (1, 100, 0)], [(0, 4, 96), (4, 7, 64)], 2, 64, 16, "head", cache16, wide=wide)
    for b in (0, 1, 4):
        c.table[b] = -1
        c.lens[b] = 0
    c.upload()
    c.h["lens"] = dev.put(c.lens)
    check(dev, rng, c, 4, act16)


@pytest.mark.parametrize("act16,cache16", TYPES)
def test_groups_and_prefixes_that_are_none(dev, act16, cache16):
    """Numbers out of range count as its nearest end: the result is the definition's whatever they say, as long as what is said to be shared is."""
    rng = np.random.default_rng(18)
    nan, inf = np.nan, np.inf
    c = Shared(dev, rng, [(1, 100, 0), (2, 90, 0), (1, 99, 0), (20, 85, 0)], [(0, 4, 64)], 2, 64, 16, "head", cache16, pad=1)
    q = rounded(rng.standard_normal((c.tokens, 4, 64)), act16)
    first = check(dev, rng, c, 4, act16, q=q)
    for groups, shared in (([0, 4], [nan]), ([0, 4], [-5.0]), ([0, 4], [64.9]), ([nan, 4], [64]), ([-3, 1e9], [64]), ([0, inf], [64]), ([4, 4], [64]), ([0, nan], [64]), ([3, 1], [64]),
                           ([0, 2, 4], [64, 50]), ([0, 3, 1, 4], [64, 64, 64]), ([2, 2, 2, 4], [0, 64, 64]), ([0, 1, 2, 3, 4], [64, 80, 64, 48])):
        c.h["groups"], c.h["shared"] = dev.put(np.float32(groups)), dev.put(np.float32(shared))
        c.groups = [0] * len(shared)
        got = check(dev, rng, c, 4, act16, q=q)
        if groups == [0, 4] and shared == [64.9]:
            assert np.array_equal(got, first)


@pytest.mark.parametrize("act16,cache16", TYPES)
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_values_that_are_not_finite(dev, act16, cache16, bad):
    """In one sequence's own positions they are no other sequence's; in the prefix they are everybody's of the group, and nobody else's; in positions of a chunk that come
    later, no earlier token's."""
    H, kvH, hs, seqs, groups = 4, 2, 64, [(1, 100, 0), (30, 140, 0), (2, 90, 0), (1, 70, 0)], [(0, 3, 64)]
    rng = np.random.default_rng(19)
    c = Shared(dev, rng, seqs, groups, kvH, hs, 16, "head", cache16)
    q = rounded(rng.standard_normal((c.tokens, H, hs)), act16)
    want, tol = attention(c, q, H, act16, None, act16)

    def run():
        c.upload()
        hq, hy = dev.put(q, act16), dev.zeros(q.size, act16)
        c.attend_shared(hq, hy, H)
        return dev.get(hy, q.shape)

    # the second sequence's token at position 130, one of its 30 new ones
    keep = c.v.copy()
    c.v[int(c.table[1, 130 // 16]), :, 130 % 16, 5] = bad
    got, touched = run(), np.zeros(c.tokens, bool)
    touched[1 + 20:31] = True
    assert (abs(got - want)[~touched] <= tol[~touched]).all()
    assert not np.isfinite(got[touched]).all(axis=(1, 2)).any()
    # a value of the prefix
    c.v[:] = keep
    c.v[int(c.table[0, 1]), :, 3, 7] = bad
    got, touched = run(), np.arange(c.tokens) < 33
    assert (abs(got - want)[~touched] <= tol[~touched]).all()
    assert not np.isfinite(got[touched][:, :, 7]).any()
    c.v[:] = keep
    # a query that is no number spoils its own row alone
    q[5, 2, 9] = np.nan
    got, touched = run(), np.zeros((c.tokens, H), bool)
    touched[5, 2] = True
    assert (abs(got - want)[~touched] <= tol[~touched]).all() and np.isnan(got[5, 2]).all()


@pytest.mark.parametrize("act16,cache16", TYPES)
@pytest.mark.parametrize("where", ["prefix", "own"])
def test_scores_that_are_all_minus_infinity_on_one_side(dev, act16, cache16, where):
    """Keys of -inf in all of the prefix, or in all of what is behind it, are weights of zero beside the other side's."""
    rng = np.random.default_rng(20)
    H, kvH, hs = 2, 1, 64
    c = Shared(dev, rng, [(1, 100, 0), (1, 90, 0), (20, 110, 0)], [(0, 3, 64)], kvH, hs, 16, "pos", cache16)
    span = (lambda m: range(64)) if where == "prefix" else (lambda m: range(64, m))
    for b, (n, m, _) in enumerate(c.seqs):
        for t in span(m):
            c.k[int(c.table[b, t // 16]), :, t % 16] = -np.inf
    c.upload()
    q = rounded(abs(rng.standard_normal((c.tokens, H, hs))) + 0.1, act16)
    hq, hy = dev.put(q, act16), dev.zeros(q.size, act16)
    c.attend_shared(hq, hy, H)
    got = dev.get(hy, q.shape)
    at = 0
    for (n, m, _), (k, v) in zip(c.seqs, c.dense):
        for j in range(n):
            seen = np.arange(64, m - n + j + 1) if where == "prefix" else np.arange(64)
            for h in range(H):
                kk, vv = k[seen, 0].astype(np.float64), v[seen, 0].astype(np.float64)
                s = kk @ q[at + j, h] / 8
                e = np.exp(s - s.max())
                w = e / e.sum()
                off = 2 * ((hs + 8) * U32 * (abs(kk) @ abs(q[at + j, h])).max() / 8 + 4 * U32 * abs(s - s.max()).max() + 4 * U32) + (2 * U16 if act16 else 0) + (len(w) + 8) * U32
                assert (abs(got[at + j, h] - w @ vv) <= off * (w @ abs(vv)) + (U16 if act16 else U32) * abs(w @ vv)).all()
        at += n


@pytest.mark.parametrize("act16,cache16", TYPES)
def test_the_same_as_attention_over_pages(dev, act16, cache16):
    """One step after another: the call's result is attention over the same pages, to both ones' tolerance, whatever was called before."""
    rng = np.random.default_rng(21)
    for H, kvH, hs, seqs, groups in ((8, 2, 128, [(1, 400 + 3 * b, 0) for b in range(20)], [(0, 20, 384)]), (4, 4, 64, [(3, 70, 0), (1, 66, 0)], [(0, 2, 48)]),
                                     (8, 2, 128, [(9, 500 + 3 * b, 0) for b in range(20)], [(0, 7, 384), (7, 20, 400)])):
        c = Shared(dev, rng, seqs, groups, kvH, hs, 16, "head", cache16)
        q = rounded(rng.standard_normal((c.tokens, H, hs)), act16)
        hq, hy, hz = dev.put(q, act16), dev.zeros(q.size, act16), dev.zeros(q.size, act16)
        c.attend_shared(hq, hy, H)
        c.attend(hq, hz, H)
        want, tol = attention(c, q, H, act16, None, act16)
        assert (abs(dev.get(hy, q.shape) - want) <= tol).all() and (abs(dev.get(hz, q.shape) - want) <= tol).all()


def test_without_scratch_memory(dev, monkeypatch):
    """Every sequence reads its pages for itself then, a workgroup a token and head."""
    rng = np.random.default_rng(31)
    monkeypatch.setenv("MYCAFFE_HIP_SCRATCH_LIMIT", "20000")
    small = Dev()
    c = Shared(small, rng, [(1, 90, 0), (3, 100, 0), (1, 70, 0), (2, 80, 0)], [(0, 3, 64)], 2, 64, 16, "head", False)
    check(small, rng, c, 4, False)
    small.close()


def test_two_kernel_objects_in_turn(dev):
    """Each has scratch memory of its own."""
    rng = np.random.default_rng(32)
    other = Dev()
    cases = [Shared(d, rng, [(1, 500 + 9 * b, 0) for b in range(12)], [(0, 12, 400 + 16 * i)], 2, 128, 16, "pos", True) for i, d in enumerate((dev, other))]
    q = [rounded(rng.standard_normal((12, 8, 128)), True) for _ in cases]
    put = [(c.dev.put(v, True), c.dev.zeros(v.size, True)) for c, v in zip(cases, q)]
    for _ in range(3):
        for c, (hq, hy) in zip(cases, put):
            c.attend_shared(hq, hy, 8)
    for c, v, (_, hy) in zip(cases, q, put):
        want, tol = attention(c, v, 8, True, None, True)
        assert (abs(c.dev.get(hy, v.shape) - want) <= tol).all()
    other.close()


@pytest.mark.parametrize("act16,cache16", TYPES)
@pytest.mark.parametrize("max_new", [1, 40, 500])
def test_hint(dev, act16, cache16, max_new):
    """The bound on new tokens changes nothing but kernels, even where it does not hold."""
    rng = np.random.default_rng(10)
    c = Shared(dev, rng, [(40, 90, 0), (1, 70, 0), (33, 83, 0)], [(0, 3, 48)], 2, 64, 16, "pos", cache16)
    check(dev, rng, c, 4, act16, max_new=max_new)


def test_refusals(dev):
    B, N, H, kvH, hs, pages, page, width = 2, 3, 4, 2, 64, 5, 16, 2
    q, y = dev.zeros(N * H * hs), dev.zeros(N * H * hs)
    n = pages * kvH * page * hs
    k, v = dev.zeros(n), dev.zeros(n)
    table, starts, lens, groups, shared = dev.zeros(B * width), dev.zeros(B + 1), dev.zeros(B), dev.zeros(3), dev.zeros(2)
    good = [B, N, H, kvH, hs, pages, page, width, q, k, v, table, starts, lens, y, kvH * page * hs, page * hs, hs, 2, groups, shared]
    names = "B N H kvH hs pages page width q k v table starts lens y sP sH sT groups hGroups hShared".split()
    f = dev.cuda.AttnPagedPrefixForward
    f(*good)

    def bad(code, **change):
        a = list(good)
        for name, value in change.items():
            a[names.index(name)] = value
        refused(code, f, *a)
    for name in names[:8]:
        bad(90001, **{name: 0})
        bad(90001, **{name: 1 << 40})
    for value in (0, -1, 3, 1 << 40):
        bad(90001, groups=value)
    bad(90010, hGroups=dev.zeros(2))
    bad(90010, hShared=dev.zeros(1))
    bad(90012, hGroups=dev.zeros(3, True))
    bad(90012, hShared=dev.zeros(2, True))
    bad(90001, hGroups=y)
    bad(90001, hShared=y)
    for name in ("q", "k", "v"):
        bad(90001, y=good[names.index(name)])
    refused(90001, f, *good, nMaxNew=-1)
    from mycaffe_amd.cudadnn import CudaDnnError
    for name in ("hGroups", "hShared", "y"):
        for h in (0, 9999):
            with pytest.raises(CudaDnnError):
                a = list(good)
                a[names.index(name)] = h
                f(*a)
