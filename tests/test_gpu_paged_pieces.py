"""ATTN_PAGED_PREFIX_FWD for long chunks: tiles of 256 rows whose positions are done in pieces (csrc/attn_paged_pipe.hip), against the definition in 64 bits at some of the heads."""
import types

import numpy as np
import pytest

from tests.test_gpu_paged import attention, rounded
from tests.test_gpu_paged_prefix import Shared

pytestmark = pytest.mark.gpu

# head size, heads, key heads, page, order, [(new, positions, dropped)], groups, padding rows: from 128 tiles on (192 at size 64), three, two, three and four pieces; sequences
# too short for as many
CASES = [(128, 64, 8, 24, "pos", [(110, 4500, 0), (128, 4700, 0), (97, 3900, 0), (110, 600, 0), (110, 4444, 0)], [(0, 3, 3000), (3, 5, 0)], 2),
         (64, 64, 8, 16, "head", [(200, 4300, 0), (210, 5000, 0), (201, 4200, 0), (190, 4100, 0)], [(0, 4, 4000)], 0),
         (128, 32, 8, 64, "head", [(256, 5000, 1024), (200, 4600, 1024), (1, 4500, 1024), (300, 4700, 1024), (333, 4800, 1024)], [(0, 5, 4096)], 1),
         (128, 32, 8, 16, "pos", [(256, 4300 + 10 * b, 0) for b in range(4)] + [(250, 2600, 0), (255, 1700, 0)], [(0, 6, 1024)], 0)]


def check(dev, rng, c, H, scale=0.0, heads=5):
    q = rounded(rng.standard_normal((c.tokens, H, c.hs)) * 1.5, True)
    hq, hy = dev.put(q, True), dev.put(np.full(q.size, 7.0, np.float32), True)
    got = []
    for _ in range(2):
        c.attend_shared(hq, hy, H, fScale=scale)
        got.append(dev.get(hy, q.shape))
    assert np.array_equal(got[0], got[1])
    live = sum(n for n, _, _ in c.seqs)
    assert np.isfinite(got[0][:live]).all() and (got[0][live:] == 7.0).all()
    for h in rng.choice(H, heads, replace=False):
        kh = h // (H // c.kvH)
        one = types.SimpleNamespace(kvH=1, hs=c.hs, tokens=c.tokens, seqs=c.seqs, dense=[(k[:, kh:kh + 1], v[:, kh:kh + 1]) for k, v in c.dense], holes=getattr(c, "holes", {}))
        want, tol = attention(one, q[:, h:h + 1], 1, True, scale or None, True)
        worst = (abs(got[0][:live, h:h + 1] - want[:live]) - tol[:live]).max()
        assert worst <= 0, "head %d: off by %.3g more than the roundings" % (h, worst)


@pytest.mark.parametrize("scale", [0.0, -0.125, 2.0])       # 2.0: scores far above those of a row's first keys, tiles that are done again
@pytest.mark.parametrize("hs,H,kvH,page,order,seqs,groups,pad", CASES)
def test_pieces(dev, hs, H, kvH, page, order, seqs, groups, pad, scale):
    rng = np.random.default_rng(40)
    check(dev, rng, Shared(dev, rng, seqs, groups, kvH, hs, page, order, True, wide=False, pad=pad, width=6200 // page + 1), H, scale)


@pytest.mark.parametrize("at", [1200, 3300, 4400])
def test_a_hole_in_one_sequence(dev, at):
    """Its tiles are done again, the others' are not."""
    rng = np.random.default_rng(41)
    hs, H, kvH, page, order, seqs, groups, pad = CASES[0]
    c = Shared(dev, rng, seqs, [(0, 3, 1000), (3, 5, 0)], kvH, hs, page, order, True, wide=False, pad=pad, width=6200 // page + 1)
    c.table[1, at // page] = -1
    c.holes = {1: [(at // page * page, at // page * page + page)]}
    c.upload()
    check(dev, rng, c, H, heads=3)
