"""CPU: the division of a ragged batch's attention over CTAs.  The header that the kernel uses is compiled for the host and
every CTA's walk is replayed: each key tile of each item is taken exactly once, in order, and the pieces of a cut item agree
on how many they are, on their order and on who they belong to."""
import ctypes
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "inferno_b200", "csrc")

SOURCE = r"""
#include <map>
#include <tuple>
#include <vector>
#include "ragged_parts.h"

struct Piece { int cta, kt0, kt1, pieces, ordinal, group; };

// 0: every tile once and the pieces consistent; otherwise the number of the check that failed.  most: the largest and the
// mean part, in the header's units of cost.
extern "C" int check(int batch, const int* n, const int* past, int heads, int T, int few, int window, int grid, double* most) {
    long long total = 0;
    std::vector<long long> at(batch);
    for (int b = 0; b < batch; ++b) {
        const RaggedHead h(n[b], past[b], T, few, window);
        long long sum = 0;
        for (int i = 0; i < h.items; ++i) {
            if (h.before(i) != sum) return 1;
            sum += h.cost(i);
        }
        if (h.total() != sum) return 2;
        at[b] = total;
        total += heads * sum;
    }
    const RaggedLine line(total, grid);
    const int parts = line.parts;
    if (parts > grid || (parts && (line.cut(0) != 0 || line.cut(parts) != total))) return 3;
    std::map<std::tuple<int, int, int>, std::vector<Piece>> got;
    double largest = 0;
    for (int c = 0; c < parts; ++c) {
        int begin[4] = {batch, 0, 0, 0}, end[4] = {batch, 0, 0, 0}, cut[2][3] = {{1, 0, 0}, {1, 0, 0}};
        for (int e = 0; e < 2; ++e) {
            const long long x = line.cut(c + e);
            for (int b = 0; b < batch; ++b) {
                const RaggedHead h(n[b], past[b], T, few, window);
                if (x >= at[b] && x < at[b] + heads * h.total()) {
                    int* out = e ? end : begin;
                    out[0] = b;
                    const RaggedPlace at_x(h, at[b], x);
                    out[1] = at_x.kvh;
                    out[2] = at_x.i;
                    out[3] = at_x.tile_of(h, line, c + e);
                    int inside = 0, first = 0;
                    for (int k = at_x.first_cut(line); k <= parts && line.cut(k) < at_x.end; ++k) {
                        const int t = at_x.tile_of(h, line, k);
                        if (t > h.first_tile(at_x.i) && t < h.end_tile(at_x.i)) {
                            if (inside++ == 0) first = k;
                            if (k != first + inside - 1) return 9;  // the cuts inside an item follow one another
                        }
                    }
                    cut[e][0] = inside + 1;
                    cut[e][1] = c - (first - 1);
                    cut[e][2] = first - 1;
                }
            }
        }
        double mine = 0;
        bool first = true;
        int cut_items = 0;
        for (int b = begin[0], kvh = begin[1], i = begin[2];;) {
            if (b >= batch) break;
            const RaggedHead h(n[b], past[b], T, few, window);
            if (i >= h.items) { i = 0; if (n[b] == 0 || ++kvh >= heads) { kvh = 0; ++b; } continue; }
            const std::tuple<int, int, int> here(b, kvh, i), last(end[0], end[1], end[2]);
            if (here > last) break;
            Piece p{c, first ? begin[3] : h.first_tile(i), here == last ? end[3] : h.end_tile(i), 1, 0, 0};
            if (first || here == last) { const int* k = first ? cut[0] : cut[1]; p.pieces = k[0]; p.ordinal = k[1]; p.group = k[2]; }
            if (p.kt0 < p.kt1) {
                got[here].push_back(p);
                mine += RAGGED_ITEM_COST + h.weight(i) * (p.kt1 - p.kt0) * RAGGED_TILE;
                if (p.pieces > 1 && ++cut_items > 2) return 4;
            }
            first = false;
            ++i;
            if (here == last) break;
        }
        if (mine > largest) largest = mine;
    }
    for (int b = 0; b < batch; ++b) {
        const RaggedHead h(n[b], past[b], T, few, window);
        for (int kvh = 0; kvh < heads; ++kvh)
            for (int i = 0; i < h.items; ++i) {
                const std::vector<Piece>& v = got[std::make_tuple(b, kvh, i)];
                int kt = h.first_tile(i);
                for (size_t k = 0; k < v.size(); ++k) {
                    if (v[k].kt0 != kt) return 5;
                    kt = v[k].kt1;
                    if (v[k].pieces != (int)v.size()) return 6;
                    if (v.size() > 1 && (v[k].ordinal != (int)k || v[k].group + v[k].ordinal != v[k].cta)) return 7;
                }
                if (kt != h.end_tile(i)) return 8;
            }
    }
    most[0] = largest;
    most[1] = parts ? (double)total / parts : 0;
    return 0;
}
"""


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    d = tmp_path_factory.mktemp("parts")
    (d / "parts.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", CSRC, str(d / "parts.cpp"), "-o", str(d / "parts.so")],
                   check=True)
    lib = ctypes.CDLL(str(d / "parts.so"))

    def run(past, new, heads, T, window, grid, few=4):
        ints = lambda v: (ctypes.c_int * len(v))(*v)  # noqa: E731
        most = (ctypes.c_double * 2)()
        rc = lib.check(len(new), ints(new), ints(past), heads, T, few, window, grid, most)
        assert rc == 0, f"check {rc} failed for past={past[:20]} new={new[:20]} heads={heads} T={T} window={window} grid={grid}"
        return most[0], most[1]

    return run


@pytest.mark.parametrize("seed", range(40))
def test_every_tile_is_taken_once(check, seed):
    rng = random.Random(seed)
    for _ in range(20):
        batch = rng.choice([1, 1, 2, 3, 17, 60])
        new = [rng.choice([0, 1, 1, rng.randint(1, 8), rng.randint(0, 300), rng.randint(0, 5000) if batch < 4 else 2]) for _ in range(batch)]
        past = [rng.choice([0, 1, 127, 128, rng.randint(0, 500), rng.randint(0, 40000)]) for _ in range(batch)]
        check(past, new, rng.choice([1, 2, 8]), rng.choice([2, 16, 32, 42, 256]), rng.choice([0, 0, 1, 100, 512, 4096]), rng.choice([1, 7, 148]),
              rng.choice([0, 1, 10]))


@pytest.mark.parametrize("past,new", [([(1 << 29) - 1], [1]), ([(1 << 29) - 300], [300]), ([0], [1 << 20]), ([0, 0], [0, 0])])
def test_extremes(check, past, new):
    check(past, new, 8 if new[0] < 1000 else 1, 42, 0, 148)
    check(past, new, 8 if new[0] < 1000 else 1, 42, 512, 148)


def test_parts_are_even(check):
    """No CTA has more than the mean part, a tile for each end of it and the fixed cost of a second piece."""
    rng = random.Random(3)
    for _ in range(20):
        new = [rng.choice([1, 1, 1, 6, rng.randint(1, 2000)]) for _ in range(30)]
        past = [rng.randint(0, 16000) for _ in range(30)]
        largest, mean = check(past, new, 8, 42, 0, 148)
        assert largest <= 1.35 * mean + 4 * 4 * 128
