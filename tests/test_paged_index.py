"""What the paged kernels take from device memory (csrc/paged.h), on the host: every number ends inside its range, whatever it is."""
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROGRAM = """
#include <cstdio>
#include <cstring>
#include "paged.h"
static float bits(unsigned u) { float f; memcpy(&f, &u, 4); return f; }
int main()
{
    char what;
    unsigned u, v, w;
    int a, b;
    while (scanf(" %c", &what) == 1) {
        if (what == 'i') { scanf("%x %d %d", &u, &a, &b); printf("%d\\n", mch::paged_int(bits(u), a, b)); }
        else if (what == 'p') { scanf("%x %d", &u, &a); printf("%d\\n", mch::paged_page(bits(u), a)); }
        else if (what == 'r') {      // total, most, least: W, every run's begin, whose every unit is, where every workgroup goes
            int least;
            scanf("%d %d %d", &a, &b, &least);
            const mch::PagedRuns r(a, b, least);
            printf("%d ", r.W);
            for (int i = 0; i <= r.W; i++) printf("%d ", r.W ? r.begin(i) : 0);
            for (int i = 0; i < a; i++) printf("%d ", r.of(i));
            for (int i = 0; i < b; i++) printf("%d ", mch::paged_place(i, r.W));
            printf("\\n");
        } else if (what == 't') {    // before, perTile, tiles, shift: units before every tile, the tile of every unit
            int tiles, shift;
            scanf("%d %d %d %d", &a, &b, &tiles, &shift);
            for (int i = 0; i <= tiles; i++) printf("%d ", mch::paged_units_before(a, b, i, shift));
            for (int i = 0; i < mch::paged_units_before(a, b, tiles, shift); i++) printf("%d ", mch::paged_tile_of(a, b, tiles, shift, i));
            printf("\\n");
        } else {
            scanf("%x %x %x %d %d", &u, &v, &w, &a, &b);
            const mch::PagedSpan s = mch::paged_span(bits(u), bits(v), bits(w), a, b);
            printf("%d %d %d\\n", s.first, s.count, s.len);
        }
    }
}
"""
BAD = [np.nan, -np.nan, np.inf, -np.inf, -1.0, -0.0, -0.5, 0.0, 0.99, 1.0, 1e-45, 3.0, 4.0, 4.5, 16777215.0, 16777216.0, 2147483648.0, 4294967296.0, 1e38, -1e38]


def hexof(v):
    return "%08x" % int(np.float32(v).view(np.uint32))


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged_index")
    (d / "main.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "mycaffe_amd", "csrc"), str(d / "main.cpp"), "-o", str(d / "main")], check=True)

    def run(lines):
        out = subprocess.run([str(d / "main")], input="\n".join(lines) + "\n", capture_output=True, text=True, check=True).stdout
        return [tuple(int(x) for x in line.split()) for line in out.splitlines()]
    return run


def test_whole_numbers(ask):
    for hi in (0, 1, 5, 1 << 24):
        got = ask(["i %s 0 %d" % (hexof(v), hi) for v in BAD])
        want = [0 if np.isnan(v) else int(min(max(np.trunc(np.float64(np.float32(v))), 0), hi)) for v in BAD]
        assert [g[0] for g in got] == want


def test_pages(ask):
    for pages in (1, 4, 1 << 24):
        got = ask(["p %s %d" % (hexof(v), pages) for v in BAD])
        want = [int(v) if v >= 0 and v < pages else -1 for v in BAD]
        assert [g[0] for g in got] == want


def test_spans_stay_inside(ask):
    triples = [(a, b, c) for a in BAD for b in BAD for c in BAD[:14]]
    for (a, b, c), (first, count, length) in zip(triples, ask(["s %s %s %s 7 40" % (hexof(a), hexof(b), hexof(c)) for a, b, c in triples])):
        assert 0 <= first and 0 <= count and first + count <= 7 and 0 <= length <= 40, (a, b, c)
    assert ask(["s %s %s %s 7 40" % (hexof(2), hexof(5), hexof(9))]) == [(2, 3, 9)]


def test_runs_cover_the_list(ask):
    """Every unit in one run, runs equal to one, no shorter than asked where there are several; places of workgroups: all runs once, neighbours on an XCD."""
    cases = [(t, m, l) for t in (0, 1, 7, 8, 63, 64, 1000, 4097) for m in (1, 7, 8, 512) for l in (1, 8)]
    for (total, most, least), out in zip(cases, ask(["r %d %d %d" % c for c in cases])):
        W, rest = out[0], out[1:]
        assert W == min(most, max(total // least, 1 if total else 0))
        begins, owners, places = rest[:W + 1], rest[W + 1:W + 1 + total], rest[W + 1 + total:]
        if W:
            sizes = np.diff(begins)
            assert begins[0] == 0 and begins[-1] == total and sizes.min() >= 1 and sizes.max() - sizes.min() <= 1
            assert sizes.min() >= least or W == 1
            assert list(owners) == list(np.repeat(np.arange(W), sizes))
        assert len(places) == most
        used = [p for p in places if p >= 0]
        assert sorted(used) == list(range(W))
        for x in range(8):
            mine = [p for p in places[x::8] if p >= 0]
            assert mine == list(range(mine[0], mine[0] + len(mine))) if mine else True


def test_tiles_of_units(ask):
    cases = [(b, p, t, s) for b in (0, 1, 5000) for p in (1, 18, 128) for t in (1, 2, 9) for s in (0, 3)] + [((1 << 24) - 5, 128, 3, 20)]
    for (before, per, tiles, shift), out in zip(cases, ask(["t %d %d %d %d" % c for c in cases])):
        starts, owner = np.array(out[:tiles + 1]), out[tiles + 1:]
        assert starts[0] == 0 and (np.diff(starts) >= 1).all()
        assert list(owner) == list(np.repeat(np.arange(tiles), np.diff(starts)))
        # about a unit for 32 << shift positions and one for the tile
        want = [(before + (i + 1) * per) / (32 << shift) + 1 for i in range(tiles)]
        assert (abs(np.diff(starts) - want) <= 1).all()
