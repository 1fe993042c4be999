"""Weights of attention behind shared prefixes (ATTN_PAGED_PREFIX_FWD, csrc/attn_prefix.hip) have sixteen bits, as single tokens over pages have them: the tolerance of 16-bit rows
without the eight bits of long chunks."""
import numpy as np
import pytest

from tests.test_gpu_paged import Cache, attention, rounded
from tests.test_gpu_paged_prefix import Shared

pytestmark = pytest.mark.gpu

# H, kvH, hs, page, order, [(new, positions, dropped)], [(first, end, shared)]: groups of more than sixteen rows, whose prefix is one product of all of them
CASES = {
    "unshared_heads": (4, 4, 64, 16, "head", [(1, 130 + b % 40, 0) for b in range(24)], [(0, 24, 128)]),
    "shared_heads": (8, 2, 128, 16, "pos", [(1, 200 + 3 * b, 0) for b in range(20)], [(0, 20, 192)]),
    "two_groups": (8, 2, 64, 8, "head", [(1 + b % 2, 100 + b, 0) for b in range(30)], [(0, 15, 96), (15, 30, 64)]),
    "size_48": (6, 3, 48, 16, "pos", [(1, 90 + b, 0) for b in range(20)], [(0, 20, 80)]),
    "chunks_of_their_own": (8, 1, 64, 16, "head", [(3, 150 + b, 0) for b in range(12)], [(0, 12, 64)]),
}


@pytest.mark.parametrize("name", CASES)
def test_weights_of_sixteen_bits(dev, name):
    H, kvH, hs, page, order, seqs, groups = CASES[name]
    rng = np.random.default_rng(len(name))
    c = Shared(dev, rng, seqs, groups, kvH, hs, page, order, True)
    # queries so small that scores, and what rounds them, are: all positions weigh about the same
    q = rounded(0.1 * rng.standard_normal((c.tokens, H, hs)), True)
    hq, hy = dev.put(q, True), dev.zeros(q.size, True)
    c.attend_shared(hq, hy, H)
    got = dev.get(hy, q.shape)
    want, tol = attention(c, q, H, False, None, True)
    # a weight is the sum of a bf16 number and one of what that leaves, 2^-8 of 2^-8 of it off; the sum of the weights is that of fp32 numbers
    sizes = Cache.__new__(Cache)
    sizes.__dict__.update(c.__dict__)
    sizes.dense = [(k, abs(v)) for k, v in c.dense]
    total, _ = attention(sizes, q, H, False)
    tol = tol + 2.0 ** -16 * total
    assert (abs(got - want) <= tol).all(), "off by %.3g of the allowance" % (abs(got - want) / tol).max()
    # and what eight bits leave of them, half of it where they are rounded at random, would be seen in values near zero
    small = abs(want) < 2.0 ** -6 * total
    assert small.any() and (tol[small] < 2.0 ** -12 * total[small]).all()
