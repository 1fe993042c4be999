"""What the host checks before a step's plan and a draw (csrc/paged.h), and the definitions that they are tested against, without a device."""
import os
import subprocess

import numpy as np
import pytest

from oracle import serving_ref as S

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROGRAM = """
#include <cstdio>
#include "paged.h"
int main()
{
    char what;
    long long l[5], at[mch::PLAN_OPERANDS];
    int n;
    while (scanf(" %c", &what) == 1) {
        for (int i = 0; i < 5; i++) scanf("%lld", l + i);
        if (what == 'z') { scanf("%d", &n); printf("%d\\n", (int)mch::plan_sizes_ok(l, n != 0)); }
        else if (what == 's') printf("%d\\n", (int)mch::sample_sizes_ok(l[0], l[1], l[2], l[3], l[4]));
        else if (what == 'v') { for (int i = 0; i < mch::PLAN_OPERANDS; i++) printf("%lld ", mch::plan_values(l, i)); printf("\\n"); }
        else {
            for (int i = 0; i < mch::PLAN_OPERANDS; i++) scanf("%lld", at + i);
            printf("%d\\n", (int)(mch::plan_clash(l, [&](int i) { return (const void*)at[i]; }, 4) != nullptr));
        }
    }
}
"""
MOST = 1 << 24


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    d = tmp_path_factory.mktemp("serving_sizes")
    (d / "main.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "mycaffe_amd", "csrc"), str(d / "main.cpp"), "-o", str(d / "main")], check=True)

    def run(*lines):
        out = subprocess.run([str(d / "main")], input="\n".join(" ".join(str(v) for v in line) for line in lines) + "\n", capture_output=True, text=True, check=True).stdout
        return [tuple(int(x) for x in line.split()) for line in out.splitlines()]
    return run


def test_sizes_of_a_plan(ask):
    good = [3, 20, 50, 16, 7]
    assert ask(["z"] + good + [1]) == [(1,)]
    assert ask(*[["z"] + good[:i] + [v] + good[i + 1:] + [0] for i in range(5) for v in (0, -1, MOST + 1, 1 << 62)]) == [(0,)] * 20
    # positions of a sequence are whole numbers of fp32, and slots too where they are asked for
    assert ask(["z", 1, 1, 1, 1 << 12, 1 << 12, 0], ["z", 1, 1, 1, 1 << 12, (1 << 12) + 1, 0], ["z", 1, 1, 1 << 20, 16, 1, 1],
               ["z", 1, 1, (1 << 20) + 1, 16, 1, 1], ["z", 1, 1, (1 << 20) + 1, 16, 1, 0]) == [(1,), (0,), (1,), (0,), (1,)]
    assert ask(["v"] + good) == [(3, 3, 21, 51, 3, 21, 51, 4, 20, 20, 3, 3, 3, 3)]


def test_where_the_operands_of_a_plan_lie(ask):
    sizes = [3, 20, 50, 16, 7]
    values = ask(["v"] + sizes)[0]
    apart = [4096 + 1024 * i for i in range(14)]
    inplace = list(apart)
    for a, b in ((1, 4), (2, 5), (3, 6), (12, 13)):
        inplace[b] = inplace[a]
    clash = lambda at: ask(["c"] + sizes + at)[0][0]  # noqa: E731
    assert not clash(apart) and not clash(inplace)
    assert not clash(inplace[:8] + [0, 0] + inplace[10:]) and not clash(inplace[:11] + [0, 0, 0])
    for a, b in ((1, 4), (2, 5), (3, 6), (12, 13)):      # one in place and the others not, one not and the others in place
        one, other = list(apart), list(inplace)
        one[b], other[b] = one[a], apart[b]
        assert clash(one) and clash(other)
    for out in (4, 5, 6, 7, 8, 9, 10, 13):
        for other in range(14):
            if other == out:
                continue
            for at in (apart[other], apart[other] + 4 * (values[other] - 1), apart[other] - 4 * (values[out] - 1)):
                assert clash(apart[:out] + [at] + apart[out + 1:]), (out, other)
            for at in (apart[other] + 4 * values[other], apart[other] - 4 * values[out]):
                assert not clash(apart[:out] + [at] + apart[out + 1:]), (out, other)
    # inputs may share memory with each other
    assert not clash([apart[1]] + apart[1:]) and not clash(apart[:11] + [apart[0]] + apart[12:])


def test_sizes_of_a_draw(ask):
    most = 1 << 20
    good = [4, 100, 4, 100, most]
    assert ask(["s"] + good, ["s", MOST, most, MOST, 1 << 38, most]) == [(1,), (1,)]
    bad = [(0, v) for v in (0, -1, MOST + 1)] + [(1, v) for v in (0, -1, 101, most + 1)] + [(2, v) for v in (0, -1, MOST + 1)] + [(3, v) for v in (0, 99, (1 << 38) + 1, -100)]
    assert ask(*[["s"] + good[:i] + [v] + good[i + 1:] for i, v in bad]) == [(0,)] * len(bad)


def test_plan_by_hand():
    table = [[0, 1, -1], [2, -1, -1], [-1, -1, -1]]
    got = S.plan([1, -1, 5], [8, 3, 0], table, [3, 5, 4, 3, 0, 0, 0], 16, 4)
    # the page of the one that ends lies on top and goes first: to position 8 of the first; then 3 and 4 to the third
    assert got["lens"] == [9, 0, 5] and got["table"].tolist() == [[0, 1, 2], [-1, -1, -1], [3, 4, -1]] and got["free"][0] == 1
    assert got["starts"] == [0, 1, 1, 6] and got["positions"] == [8, 0, 1, 2, 3, 4] and got["slots"] == [8, 12, 13, 14, 15, 16] and got["last"] == [0, -1, 5]
    # the second does not fit the rows, and the third waits behind it though it would
    got = S.plan([1, 5, 1], [8, 3, 0], table, [3, 5, 4, 3, 0, 0, 0], 5, 4)
    assert got["lens"] == [9, 3, 0] and got["starts"] == [0, 1, 1, 1]
    # the third begins behind the first page of the first
    got = S.plan([1, 1, 2], [8, 3, 0], table, [3, 5, 4, 3, 0, 0, 0], 5, 4, [-1, -1, 0], [0, 0, 7])
    assert got["lens"] == [9, 4, 6] and got["table"][2].tolist() == [0, 4, -1] and got["shared"] == [0, 0, 4]


def test_draws_by_hand():
    x = np.log([1.0, 4.0, 2.0, 1.0])
    assert [S.sample(x, u)[0] for u in (0.0, 0.12, 0.13, 0.62, 0.63, 0.87, 0.88, 1.0, 7.0, -1.0)] == [0, 0, 1, 1, 2, 2, 3, 3, 3, 0]
    assert [S.sample(x, u, k=2)[0] for u in (0.0, 0.66, 0.67)] == [1, 1, 2] and [S.sample(x, u, k=3)[0] for u in (0.1, 0.2, 0.9)] == [0, 1, 2]
    assert [S.sample(x, u, p=0.6)[0] for u in (0.6, 0.7)] == [1, 2] and S.sample(x, 0.99, p=0.4)[0] == 1
    assert [S.sample(x, u, m=0.3)[0] for u in (0.6, 0.7)] == [1, 2] and S.sample(x, 0.3, temperature=0)[0] == 1
    assert S.sample([-np.inf, np.nan], 0.5)[0] == -1 and S.sample([np.inf, 3, np.inf], 0.6)[0] == 2
    assert abs(S.sample(x, 0.5)[1] - np.log(0.5)) < 1e-15
