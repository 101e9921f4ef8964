"""The host's arithmetic of linear attention's chunks (qmag_linattn_plan.h), compiled for the tests."""
import atexit
import os
import shutil
import subprocess
import tempfile

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

ASK = r"""
#include <stdio.h>
#include "qmag_linattn_plan.h"
using namespace qmag;

// stdin: calls of T n_seq n_key n_head dim_k dim_v parts; stdout: the window's rows, the workspace's bytes, and the
// rows up to which a sequence goes token by token
int main()
{
    int T, n, keys, heads, dk, dv, parts;
    while (scanf("%d%d%d%d%d%d%d", &T, &n, &keys, &heads, &dk, &dv, &parts) == 7) {
        const int brief = la_brief((int64_t)n * heads * (dv / 16), parts);
        const size_t tile = la_tile_bytes(parts, dk, keys, heads), state = (size_t)4 * heads * dk * dv;
        const int window = la_window(T, n, brief, tile, state);
        printf("%d %zu %d\n", window, window ? la_workspace(window, T, n, brief, tile, state) : (size_t)0, brief);
    }
}
"""
_exe = None


def windows(calls):
    """calls of (T, n_seq, n_key, n_head, dim_k, dim_v, parts): (rows of a window, 0 for none; bytes; brief) each."""
    global _exe
    cc = shutil.which("g++")
    if not cc:
        pytest.skip("no host compiler")
    if _exe is None:
        d = tempfile.mkdtemp(prefix="linattn_plan")
        atexit.register(shutil.rmtree, d, ignore_errors=True)
        src = os.path.join(d, "ask.cpp")
        with open(src, "w") as f:
            f.write(ASK)
        subprocess.run([cc, "-std=c++17", "-O1", "-I", os.path.join(ROOT, "qwen-mobile-agent_amd", "csrc"), src, "-o",
                        os.path.join(d, "ask")], check=True)
        _exe = os.path.join(d, "ask")
    text = "\n".join(" ".join(str(int(x)) for x in c) for c in calls)
    out = subprocess.run([_exe], input=text, capture_output=True, text=True, check=True, timeout=120).stdout.split("\n")
    return [tuple(int(x) for x in line.split()) for line in out if line]
