"""Attention behind shared prefixes as a server calls it: memory for far more rows than a step has, tables far wider than its sequences, and what it says of the step
(maxNew), right or wrong, which only chooses kernels."""
import numpy as np
import pytest

from tests.test_gpu_paged import TYPES
from tests.test_gpu_paged_prefix import Shared, check

pytestmark = pytest.mark.gpu

STEPS = {
    "single_tokens": (8, 2, 64, [(1, 200 + 7 * b, 0) for b in range(20)], [(0, 20, 192)]),
    "unshared_heads": (4, 4, 64, [(b % 4 > 0, 90 + 7 * b, 0) for b in range(24)], [(0, 10, 80), (10, 24, 64)]),
    "a_prompt_among_them": (4, 2, 128, [(1, 140 + b, 0) if b != 5 else (150, 300, 0) for b in range(12)], [(0, 12, 128)]),
}


@pytest.mark.parametrize("act16,cache16", TYPES)
@pytest.mark.parametrize("name", STEPS)
def test_room_for_more(dev, name, act16, cache16):
    H, kvH, hs, seqs, groups = STEPS[name]
    rng = np.random.default_rng(len(name))
    c = Shared(dev, rng, [(int(n), m, gone) for n, m, gone in seqs], groups, kvH, hs, 16, "head", cache16, pad=4000)
    for max_new in (1, 0, max(n for n, _, _ in c.seqs), 5000):
        check(dev, np.random.default_rng(3), c, H, act16, max_new=max_new)
