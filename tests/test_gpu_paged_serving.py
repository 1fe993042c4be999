"""Append (id 2015) and attention over pages (id 2016) call after call, as a server makes them, each held to the roundings of its own step: what the append
has stored is read back, and attention is the definition's in 64 bits over exactly that."""
import numpy as np
import pytest

from tests.test_gpu_paged import EPS, THETA, TYPES, U16, U32, attention, head_norm, pair_size, rounded, turned

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act16,cache16", TYPES)
@pytest.mark.parametrize("H,kvH,hs,page,order", [(4, 2, 64, 16, "head"), (6, 6, 48, 8, "pos"), (8, 1, 128, 24, "pos"), (4, 2, 160, 16, "head"), (3, 1, 22, 5, "pos")])
def test_calls_one_after_the_other(dev, H, kvH, hs, page, order, act16, cache16):
    """Three sequences in chunks and single tokens, pages handed out in any order as they grow, a padded batch, oldest pages given up on the way."""
    rng = np.random.default_rng(70 + hs)
    plans = [[40, 0, 3], [40, 30, 1], [0, 1, 1], [17, 1, 50], [1, 1, 1], [1, 1, 1], [1, 25, 1], [0, 1, 2], [0, 1, 1]]
    totals = [sum(p[b] for p in plans) for b in range(3)]
    width = -(-max(totals) // page) + 1
    count = sum(-(-t // page) for t in totals) + 2
    rows = [rounded(rng.standard_normal((t, H + 2 * kvH, hs)), act16) for t in totals]
    w = [rounded(1 + 0.2 * rng.standard_normal(hs), act16) for _ in range(2)]
    free, table = list(rng.permutation(count)), np.full((3, width), -1, np.float32)
    empty = np.full(count * kvH * page * hs, np.nan, np.float32)
    hk, hv = dev.put(empty, cache16), dev.put(empty, cache16)
    hr = dev.cuda.CreateRope(0, 0, 1, 1, width * page, H, hs, THETA)
    hw = [dev.put(x, act16) for x in w]
    whole = kvH * page * hs
    strides = (whole, page * hs, hs) if order == "head" else (whole, hs, kvH * hs)

    def pages_of(h):      # (pages, positions, heads, values)
        a = dev.get(h)
        return a.reshape(count, kvH, page, hs).transpose(0, 2, 1, 3) if order == "head" else a.reshape(count, page, kvH, hs)
    have, gone = [0, 0, 0], [0, 0, 0]
    stored = [tuple(np.zeros((0, kvH, hs)) for _ in range(2)) for _ in range(3)]
    # the norm: hs roundings of the mean's terms, halved by the root; root, quotient, two products; the rotation: two products, their sum, rounded cosine and sine
    off = (hs + 2) * U32 / 2 + 6 * U32 + 4 * U32
    for i, plan in enumerate(plans):
        pad = i % 3
        new = np.concatenate([rows[b][have[b]:have[b] + n] for b, n in enumerate(plan)] + [np.full((pad, H + 2 * kvH, hs), 9.0, np.float32)])
        have = [a + n for a, n in zip(have, plan)]
        for b in range(3):
            for e in range(gone[b] // page, -(-have[b] // page)):
                if table[b, e] < 0:
                    table[b, e] = free.pop()
        ht, hs_, hl = dev.put(table), dev.put(np.float32(np.concatenate([[0], np.cumsum(plan)]))), dev.put(np.float32(have))
        N, live = len(new), sum(plan)
        hq, hy = dev.put(np.full(N * H * hs, 7.0, np.float32), act16), dev.put(np.full(N * H * hs, 7.0, np.float32), act16)
        sizes = (3, N, H, kvH, hs, count, page, width)
        dev.cuda.PagedAppend(*sizes, dev.put(new, act16), hq, hk, hv, ht, hs_, hl, *strides, hr, True, *hw, EPS)
        dev.cuda.AttnPagedForward(*sizes, hq, hk, hv, ht, hs_, hl, hy, *strides)
        got, q = dev.get(hy, (N, H, hs)), dev.get(hq, (N, H, hs))
        assert (got[live:] == 7.0).all() and (q[live:] == 7.0).all()
        pk, pv = pages_of(hk), pages_of(hv)
        dense, at = [], 0
        for b, n in enumerate(plan):
            before = stored[b]
            where = [(int(table[b, t // page]) if t >= gone[b] else 0, t % page) for t in range(have[b])]
            k, v = (np.stack([p[a, s] for a, s in where]) if where else np.zeros((0, kvH, hs), np.float32) for p in (pk, pv))
            m = have[b] - n
            x, pos = rows[b][m:have[b]].astype(np.float64), np.arange(m, have[b])
            # what was there has stayed; what is new is the definition's, to the roundings of its way
            keep = slice(min(gone[b], m), m)
            assert np.array_equal(k[keep], before[0][keep]) and np.array_equal(v[keep], before[1][keep])
            for g, raw, wt, half in ((q[at:at + n], x[:, :H], w[0], act16), (k[m:], x[:, H:H + kvH], w[1], cache16)):
                plain = head_norm(raw, wt.astype(np.float64))
                want = turned(plain, pos)
                assert (abs(g - want) <= off * pair_size(plain) + (U16 if half else U32) * abs(want)).all()
            assert np.array_equal(v[m:], rounded(x[:, H + kvH:], cache16))
            stored[b] = (k, v)
            dense.append((k, v))
            at += n
        c = type("C", (), dict(kvH=kvH, hs=hs, tokens=N, seqs=[(n, m, g) for n, m, g in zip(plan, have, gone)], dense=dense))
        want, tol = attention(c, q, H, act16, None, act16)
        assert (abs(got - want)[:live] <= tol[:live]).all(), i
        if i == 3:      # the first sequence's oldest pages go, and are others' from now on
            gone[0] = 2 * page
            free += [int(p) for p in table[0, :2]]
            table[0, :2] = -1
    dev.cuda.FreeRope(hr)
