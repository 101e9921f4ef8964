"""The attention entries where forms, lengths and magnitudes meet: lengths that are
none, values far apart in size, infinite keys, the forms that only large calls take."""
import numpy as np
import pytest

from attn_fixtures import BF16, F16, F32, TYPES, View, attention, held, ints, to_type, values
from test_gpu_attn import CacheCase, check_kv4, close, kv4_tol, kv_values, rng_of, run_kv4, run_prompt

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------ lengths that are none --

@pytest.mark.parametrize("typ", ["f32", "bf16"])
@pytest.mark.parametrize("rows,n", [(4, 40), (90, 9)])
def test_attn_kv4_lengths_that_lap_over(qm, typ, rows, n):
    """cu up and down, so that sequences of several parts ask for more of them than a call has:
    some rows are left out, nothing but rows is written, and what is written is finite."""
    t = TYPES[typ]
    r = rng_of(rows, n)
    L = 1000
    case = CacheCase(qm, r, [L], 1, 64, 16)
    table = ints(qm, np.repeat(case.table, n, 0))
    c = qm.KvTable(n, case.table.shape[1], 16, case.n_block, table.ptr, None)
    q = View(qm, to_type(r.randn(rows, 8, 64), t), t, "gap")
    out = View(qm, to_type(np.full((rows, 8, 64), 3), t), t, "gap", fill=3)
    cu, lens = ints(qm, [rows * (i % 2) for i in range(n + 1)]), ints(qm, [L if i > n // 2 else 1 for i in range(n)])
    qm.attn_kv4_dev(case.c, c, t, q.heads, out.heads, cu.ptr, lens.ptr, rows, 0.125)
    got, rest = out.read()
    assert rest and np.isfinite(values(got, t)).all()
