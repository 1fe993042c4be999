"""Attention over pages (id 2016) of fp32 rows where numbers are as small or as large as fp32 has them, chunks and single tokens, against the definition in
64 bits.  No tolerance has an absolute part but the half steps of numbers that fp32 stores without all of their bits."""
import numpy as np
import pytest

from tests.test_gpu_paged import Cache, U32, rounded

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -149      # between the smallest numbers of fp32


def definition(c, q, H, scale):
    """y and its tolerance: roundings as the other tests of this call count them, and half a step of the smallest numbers for every product and sum"""
    G, hs, y, tol, at = H // c.kvH, c.hs, [], [], 0
    scale = scale or hs ** -0.5
    for (n, m, _), (k, v) in zip(c.seqs, c.dense):
        sees = np.arange(m)[None, :] <= np.arange(m - n, m)[:, None]
        ys, ts = np.zeros((n, H, hs)), np.zeros((n, H, hs))
        for h in range(H):
            kk, vv, qq = k[:, h // G].astype(np.float64), v[:, h // G].astype(np.float64), q[at:at + n, h].astype(np.float64)
            s = np.where(sees, scale * (qq @ kk.T), -np.inf)
            s -= s.max(1, keepdims=True)
            w = np.exp(s)
            w /= w.sum(1, keepdims=True)
            size = abs(scale) * (abs(qq) @ abs(kk).T)      # a magnitude, whatever the sign of the scale
            ds = (hs + 8) * U32 * np.where(sees, size, 0).max(1) + 4 * U32 * np.where(sees, abs(s), 0).max(1) + 4 * U32
            off = 2 * ds + (sees.sum(1) + 8) * U32
            ys[:, h] = w @ vv
            ts[:, h] = off[:, None] * (w @ abs(vv)) + U32 * abs(ys[:, h]) + (2 * sees.sum(1)[:, None] + 8) * STEP / 2
        y.append(ys)
        tol.append(ts)
        at += n
    return np.concatenate(y), np.concatenate(tol)


def check(dev, c, q, H, scale=0.0):
    for b, (k, v) in enumerate(c.dense):
        for t in range(len(k)):
            page, slot = int(c.table[b, t // c.page]), t % c.page
            c.k[page, :, slot], c.v[page, :, slot] = k[t], v[t]
    c.h["k"], c.h["v"] = dev.put(c.laid(c.k), c.half), dev.put(c.laid(c.v), c.half)
    hq, hy = dev.put(q), dev.zeros(q.size)
    c.attend(hq, hy, H, fScale=scale)
    got = dev.get(hy, q.shape)
    c.attend(hq, hy, H, fScale=scale)
    assert np.array_equal(got, dev.get(hy, q.shape))
    want, tol = definition(c, q, H, scale)
    over = abs(got - want) - tol
    at = np.unravel_index(over.argmax(), over.shape)
    assert over.max() <= 0, "%s: %g, not %g +- %g" % (at, got[at], want[at], tol[at])


# a chunk; single tokens; a chunk in many pieces; chunks and single tokens
SEQS = [[(40, 90, 0)], [(1, 90, 0), (1, 7, 0)], [(30, 3000, 0)], [(150, 333, 0), (1, 200, 0), (20, 20, 0)]]


@pytest.mark.parametrize("seqs", SEQS, ids=["chunk", "steps", "pieces", "mixed"])
@pytest.mark.parametrize("hs", [48, 64, 128])
@pytest.mark.parametrize("size", [1e-28, 1e-31, 1e-33, 1e-35, 1e-37])
@pytest.mark.parametrize("cache16", [False, True])
def test_small_values(dev, cache16, size, hs, seqs):
    """Values of this size, all of them or every third column, and one beside ordinary ones."""
    for which in ("all", "columns", "one"):
        rng = np.random.default_rng(60)
        c = Cache(dev, rng, seqs, 2, hs, 16, "head", cache16)
        for _, v in c.dense:
            small = rounded(size * np.sign(v) * (1 + abs(v)), cache16)
            if which == "all":
                v[:] = small
            elif which == "columns":
                v[:, :, ::3] = small[:, :, ::3]
            else:
                v[0, 0, 1] = small[0, 0, 1]
        check(dev, c, np.float32(rng.standard_normal((c.tokens, 4, hs))), 4)


@pytest.mark.parametrize("cache16", [False, True])
@pytest.mark.parametrize("seqs", SEQS, ids=["chunk", "steps", "pieces", "mixed"])
@pytest.mark.parametrize("hs", [64, 128])
def test_small_and_large_factors(dev, hs, seqs, cache16):
    """Scores of ordinary size whose queries are small and keys large, or the other way round."""
    for q_size, k_size in ((1e-37, 1e37), (1e37, 1e-37), (1e-34, 1e33), (1e30, 1e-31)):
        if cache16 and k_size < 1:
            continue      # 16-bit keys are multiplied as they are
        rng = np.random.default_rng(61)
        c = Cache(dev, rng, seqs, 2, hs, 16, "pos", cache16)
        for k, _ in c.dense:
            k[:] = rounded(k_size * np.sign(k) * (0.5 + 0.5 * rng.random(k.shape)), cache16)
        q = rng.standard_normal((c.tokens, 4, hs))
        check(dev, c, np.float32(q_size * np.sign(q) * (1 + 0.5 * rng.random(q.shape))), 4)


@pytest.mark.parametrize("cache16", [False, True])
def test_a_small_factor_beside_ordinary_ones(dev, cache16):
    """One key and one query of a chunk that lose bits in parts: neither has a say at ordinary sizes."""
    rng = np.random.default_rng(62)
    c = Cache(dev, rng, [(40, 90, 0), (9, 400, 0)], 2, 64, 16, "head", cache16)
    q = np.float32(rng.standard_normal((c.tokens, 4, 64)))
    q[3, 1, 5] = 1.2345e-36
    if not cache16:
        c.dense[0][0][10, 0, 7] = 3.21e-37
        c.dense[1][0][0, 1] = 0
    check(dev, c, q, 4)


@pytest.mark.parametrize("seqs", SEQS, ids=["chunk", "steps", "pieces", "mixed"])
@pytest.mark.parametrize("hs", [48, 64, 128])
def test_columns_of_zeros_and_of_the_smallest_numbers(dev, hs, seqs):
    """A column of zeros comes out as zeros, also beside one of numbers that no 16-bit part holds, which come out as they are."""
    for size in (0.0, 1e-41):
        rng = np.random.default_rng(63)
        c = Cache(dev, rng, seqs, 2, hs, 16, "head", False)
        for _, v in c.dense:
            v[:, :, 3] = 0
            if size:
                v[:, 1, hs - 1] = np.float32(size * (1 + abs(v[:, 1, hs - 1])))
        check(dev, c, np.float32(rng.standard_normal((c.tokens, 4, hs))), 4)


@pytest.mark.parametrize("cache16", [False, True])
@pytest.mark.parametrize("sign", [1, -1])
def test_small_queries_at_a_large_scale(dev, sign, cache16):
    for seqs in SEQS:
        rng = np.random.default_rng(64)
        c = Cache(dev, rng, seqs, 2, 64, 16, "head", cache16)
        check(dev, c, np.float32(1e-36 * rng.standard_normal((c.tokens, 4, 64))), 4, sign * float(np.float32(1.25e35)))
