"""CPU check of how packed sequences are cut into tiles: the arithmetic of qmag_seq.h is
compiled for the host and walked through for every tile number of a call.  Every row of
ascending sequences has exactly one tile, and whatever the sums are no tile leaves the
rows or the numbers that the host counts on."""
import os
import shutil
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

WALK = r"""
#include <stdio.h>
#include <vector>
#include "qmag_seq.h"
using namespace qmag;

// stdin: calls of T shift n_seq, then cu
int main()
{
    int T, shift, n;
    for (int call = 0; scanf("%d%d%d", &T, &shift, &n) == 3; call++) {
        std::vector<int> cu(n + 1), rows(T);
        for (int &v : cu) if (scanf("%d", &v) != 1) return 1;
        bool ascending = cu[0] >= 0 && cu[n] <= T;
        for (int i = 0; i < n; i++) ascending = ascending && cu[i] <= cu[i + 1];
        const int most = seq_most_tiles(T, n, shift);
        for (int j = 0; j < most; j++) {
            const SeqTile s = seq_find([&](int i) { return cu.at(i); }, n, T, shift, j);
            if (s.seq < 0) continue;
            if (s.seq >= n || s.tile < 0 || s.tile >= seq_tiles(s.n, shift) || s.first < 0 || s.first + s.n > T)
                return printf("call %d: tile %d is %d of sequence %d, rows %d + %d of %d\n", call, j, s.tile, s.seq, s.first, s.n, T), 1;
            if (seq_tile0(s.first, s.seq, shift) + s.tile != j) return printf("call %d: tile %d has another number\n", call, j), 1;
            for (int r = s.tile << shift; r < s.n && r < (s.tile + 1) << shift; r++) rows[s.first + r]++;
        }
        // every tile of any sequence has a number that the host counts
        for (int i = 0; i < n; i++) {
            const int a = seq_row(cu[i], T), m = seq_row(cu[i + 1], T) - a;
            if (seq_tiles(m, shift) && seq_tile0(a, i, shift) + seq_tiles(m, shift) > most)
                return printf("call %d: sequence %d ends behind the tiles\n", call, i), 1;
        }
        if (ascending)
            for (int r = 0; r < T; r++)
                if (rows[r] != (r >= cu[0] && r < cu[n])) return printf("call %d: row %d has %d tiles\n", call, r, rows[r]), 1;
    }
    return puts("ok"), 0;
}
"""


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    cc = shutil.which("g++")
    if not cc:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("seq")
    (d / "walk.cpp").write_text(WALK)
    exe = str(d / "walk")
    subprocess.run([cc, "-std=c++17", "-O1", "-D_GLIBCXX_ASSERTIONS", "-I", os.path.join(ROOT, "qwen-mobile-agent_amd", "csrc"),
                    str(d / "walk.cpp"), "-o", exe], check=True)

    def go(calls):
        text = "\n".join(" ".join(map(str, [T, shift, len(cu) - 1] + list(cu))) for T, shift, cu in calls)
        r = subprocess.run([exe], input=text, capture_output=True, text=True, timeout=300)
        assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
    return go


def test_ascending_sequences(walk):
    r = np.random.RandomState(1)
    calls = []
    for _ in range(400):
        n, shift = r.randint(1, 40), r.randint(2, 7)
        lens = r.randint(0, r.choice([2, 5, 65, 200]) + 1, n) * (r.rand(n) < 0.8)
        cu = np.concatenate([[0], np.cumsum(lens)])
        calls.append((int(cu[-1]) + r.choice([0, 0, 3]), shift, cu))
    calls += [(64 * n, 6, np.arange(n + 1) * 64) for n in (1, 2, 63)] + [(4096, 6, np.arange(4097))]
    walk(calls)


def test_sums_of_any_kind(walk):
    r = np.random.RandomState(2)
    calls = []
    for _ in range(400):
        n, shift, T = r.randint(1, 30), r.randint(2, 7), r.randint(1, 400)
        cu = r.choice([r.randint(-T, 2 * T), 0, T, -2 ** 31, 2 ** 31 - 1], n + 1) if r.rand() < 0.3 else r.randint(-9, T + 9, n + 1)
        calls.append((T, shift, cu))
    walk(calls)
