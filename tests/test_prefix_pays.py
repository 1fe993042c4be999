"""Which calls of attention behind shared prefixes share (csrc/paged.h), and what a batch on the device says of its steps, without a device."""
import os
import subprocess

import numpy as np
import pytest

from mycaffe_amd.layers import PagedBatch
from tests.test_layers_batch import Memory
from tests.test_layers_paged import attention, serve

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROGRAM = """
#include <cstdio>
#include "paged.h"
int main()
{
    long long l[8];
    while (scanf("%lld %lld %lld %lld %lld %lld %lld", l, l + 1, l + 2, l + 3, l + 4, l + 5, l + 6) == 7) {
        const long long rows = mch::prefix_rows(l[0], l[1], l[2]);
        printf("%lld %d\\n", rows, (int)mch::prefix_pays(rows, l[1], l[3], l[4], (double)l[5], l[6] != 0));
    }
}
"""


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    d = tmp_path_factory.mktemp("prefix_pays")
    (d / "main.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "mycaffe_amd", "csrc"), str(d / "main.cpp"), "-o", str(d / "main")], check=True)

    def run(tokens, batch, max_new, each=4, positions=16384, size=10 ** 9, f32=0):
        line = " ".join(str(v) for v in (tokens, batch, max_new, each, positions, size, f32))
        rows, pays = subprocess.run([str(d / "main")], input=line, capture_output=True, text=True, check=True).stdout.split()
        return int(rows), bool(int(pays))
    return run


def test_rows_are_what_the_step_can_have(ask):
    # a step of single tokens shares whatever room for prompts the memory has; where nothing is said of the step, the memory decides
    assert ask(64, 64, 0) == (64, True) and ask(64, 64, 1) == (64, True)
    assert ask(8192, 64, 1) == (64, True) and ask(8192, 64, 0) == (8192, False) and ask(8192, 64, 200) == (8192, False)
    assert ask(8192, 64, 16) == (1024, True) and ask(8192, 64, 17) == (1088, False)
    assert ask(1 << 24, 4096, 1 << 24) == (1 << 24, False)
    # too little to save, one sequence
    assert not ask(64, 64, 1, positions=2000, size=10 ** 8)[1] and ask(64, 64, 1, positions=2000, size=10 ** 8, f32=1)[1]
    assert not ask(8192, 1, 1)[1]


def test_a_step_says_how_many_tokens_it_has_at_most():
    class Told(Memory):
        def AttnPagedPrefixForward(self, *a, nMaxNew=0, **k):
            self.calls.append(("prefix", nMaxNew))

        def AttnPagedForward(self, *a, nMaxNew=0, **k):
            self.calls.append(("pages", nMaxNew))

    cuda = Told()
    batch, layer = PagedBatch(cuda, 4, 7, 6, 4, 4), attention(cuda)
    for new, said in (([1, 1, 0, 1], 1), ([1, 5, -1, 0], 5), ([-1, -1, 0, 0], 0), (None, 0), (np.array([2, 2, 2, 1.0]), 2)):
        batch.Share([0, 4], [4])
        batch.Step(new)
        serve(cuda, [layer], batch)
        assert [c for c in cuda.calls if isinstance(c, tuple)][-1] == ("prefix", said)
    batch.Share()
    batch.Step([1, 1, 1, 1])
    serve(cuda, [layer], batch)
    assert [c for c in cuda.calls if isinstance(c, tuple)][-1] == ("pages", 1)
