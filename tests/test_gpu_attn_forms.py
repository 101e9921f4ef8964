"""The forms of the attention entries that only large calls take: many parts joined by
many waves, calls that are not split, sequences far down a long list, loops over the grid."""
import numpy as np
import pytest

from attn_fixtures import BF16, F16, F32, HALF, TYPES, View, attention, held, ints, rope, to_type, values
from test_gpu_attn import (CacheCase, Pool, assign_ref, check_kv4, close, kv4_tol, kv_values, prompt_tol, rng_of, run_assign,
                           run_kv4)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------ attention over the cache --

@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("typ", TYPES)
def test_attn_kv4_many_parts(qm, typ, D):
    """One token, few heads, a table of more than 6,144 tokens: 63 to 70 parts a row, joined by 16 waves."""
    t = TYPES[typ]
    r = rng_of(D, 90)
    for L in (8000, 8999):
        case = CacheCase(qm, r, [L], 2, D, 64)
        q = to_type(r.randn(3, 4, D), t)
        check_kv4(case, q, [1], t, run_kv4(qm, case, q, [1], t))


def test_attn_kv4_a_wide_table_of_short_sequences(qm):
    """The same join where most of what the table could hold is not there."""
    for t in (F32, BF16):
        r = rng_of(91, t)
        case = CacheCase(qm, r, [300, 0, 7], 2, 128, 16, extra_cols=600)
        q = to_type(r.randn(3, 4, 128), t)
        check_kv4(case, q, [1, 1, 1], t, run_kv4(qm, case, q, [1, 1, 1], t, pad=0))


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("D,n,H", [(64, 700, 48), (128, 1030, 32), (256, 512, 32)])
def test_attn_kv4_rows_that_fill_the_chip(qm, typ, D, n, H):
    """Decode of so many rows that no sequence is split, a long one among them."""
    t = TYPES[typ]
    r = rng_of(D, n, 92)
    lens = r.randint(0, 40, n)
    lens[n // 2], lens[n - 1] = 700, 33
    case = CacheCase(qm, r, lens, 2, D, 16)
    q = to_type(r.randn(n + 2, H, D), t)
    got = run_kv4(qm, case, q, [1] * n, t)
    heads = [0, H // 2 - 1, H - 1]
    for i in range(n):
        for h in heads:
            g = h // (H // 2)
            want, mag, es = attention(values(q[i:i + 1, h:h + 1], t), case.k[i][:, g:g + 1], case.v[i][:, g:g + 1], [lens[i] - 1], D ** -0.5)
            close(values(got[i:i + 1, h:h + 1], t), want, kv4_tol(t, D, lens[i], want, mag, es), (i, h))


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("D,H", [(64, 128), (128, 128), (256, 64)])
def test_attn_kv4_chunks_that_fill_the_chip(qm, typ, D, H):
    """Two chunks of 512 rows over a cache, in the form that is not split."""
    t = TYPES[typ]
    r = rng_of(D, 93)
    lens, ask = [900, 530], [512, 512]
    case = CacheCase(qm, r, lens, 2, D, 32)
    q = to_type(r.randn(1024 + 2, H, D), t)
    got = run_kv4(qm, case, q, ask, t)
    rows = np.unique(np.concatenate([np.arange(0, 512, 37), [1, 15, 16, 127, 128, 510, 511]]))
    for i, at in ((0, 0), (1, 512)):
        for h in (0, H // 2 - 1, H - 1):
            g = h // (H // 2)
            want, mag, es = attention(values(q[at + rows, h:h + 1], t), case.k[i][:, g:g + 1], case.v[i][:, g:g + 1],
                                      lens[i] - 512 + rows, D ** -0.5)
            close(values(got[at + rows, h:h + 1], t), want, kv4_tol(t, D, lens[i], want, mag, es), (i, h))


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("n,ask", [(130, 1), (200, 1), (130, 70)])
def test_attn_kv4_long_sequences_far_down_the_list(qm, typ, n, ask):
    """More sequences than a wave takes at once, those that are split behind the first 64: their items
    and rows are found across the batches."""
    t = TYPES[typ]
    r = rng_of(n, ask, 94)
    lens = r.randint(1, 30, n)
    lens[3], lens[70], lens[n - 2] = 600, 3000, 1500
    asks = np.ones(n, int)
    if ask > 1:
        lens += ask
        asks[:] = ask
        asks[[5, 64, 90]] = 0
    case = CacheCase(qm, r, lens, 2, 64, 16)
    q = to_type(r.randn(int(asks.sum()) + 2, 2, 64), t)
    got = run_kv4(qm, case, q, asks, t)
    some = np.arange(n) if ask == 1 else [0, 3, 63, 65, 70, 71, 128, 129]
    at = np.concatenate([[0], np.cumsum(asks)])
    for i in some:
        m, L, s = int(asks[i]), int(lens[i]), slice(at[i], at[i + 1])
        want, mag, es = attention(values(q[s], t), case.k[i], case.v[i], L - m + np.arange(m), 0.125)
        close(values(got[s], t), want, kv4_tol(t, 64, L, want, mag, es), i)


# --------------------------------------------------------------------- loops over a grid --

@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("T,KV,D,bs", [(9001, 8, 128, 64), (5003, 8, 256, 16), (70001, 2, 64, 256)])
def test_append_and_read_of_long_prompts(qm, typ, T, KV, D, bs):
    """More tokens than the workgroups take at once."""
    t = TYPES[typ]
    r = rng_of(T, D)
    n_block = T // bs + 2
    k, v = (to_type(x, t) for x in (r.randn(T, KV, D).astype(np.float32) * 3 + 1, r.randn(T, KV, D).astype(np.float32)))
    slot = r.permutation(n_block * bs)[:T]
    slot[[5, T - 1]] = -1, n_block * bs
    cache = qm.DBuf.from_array(np.zeros(n_block * KV * bs * (D + D // 8), np.uint8))
    c = qm.Kv4(cache.ptr, n_block, bs, KV, D)
    kd, vd, sl = View(qm, k, t), View(qm, v, t), ints(qm, slot)
    qm.kv4_append_dev(c, t, kd.heads, vd.heads, sl.ptr, T)
    ko, vo = qm.DBuf(4 * T * KV * D), qm.DBuf(4 * T * KV * D)
    qm.kv4_read_dev(c, sl.ptr, T, ko.ptr, vo.ptr)
    live = ((slot >= 0) & (slot < n_block * bs))[:, None, None]
    for x, o in ((k, ko), (v, vo)):
        want = held(values(x, t).astype(np.float32)) * live
        assert np.array_equal(o.download(np.float32).reshape(T, KV, D).astype(np.float64), want)


def test_rope_of_a_million_tokens(qm):
    T, D = (1 << 20) + 3, 8
    r = rng_of(95)
    x, pos = r.randn(T, 1, D).astype(np.float32), r.randint(0, 5000, (2, T))
    xd, od, p = View(qm, x, F32), View(qm, np.zeros_like(x), F32), ints(qm, pos)
    qm.rope_dev(qm.Rope.make(D, D, (1, 3), True, True, 1e4), p.ptr, T, F32, xd.heads, od.heads)
    want = rope(x.astype(np.float64), pos, D, (1, 3), True, True, 1e4)
    close(od.read()[0].astype(np.float64), want, 2 * np.abs(x).max() * (2 * np.pi * 2.0 ** -26 + 5 * 2.0 ** -24))


def test_assign_of_a_million_tokens(qm):
    """More tokens than the workgroups take at once, into two sequences; then both end."""
    bs, max_blocks = 256, 4096
    held_, new = np.array([100, 0]), np.array([600000, 500001])
    T = int(new.sum()) + 5
    n_block = int((-(-(held_ + new) // bs)).sum()) + 3
    r = rng_of(96)
    order = r.permutation(n_block)
    table = np.full((2, max_blocks), -1)
    table[0, 0] = order[-1]
    free = np.concatenate([order[:-1], [-5]])
    pool = Pool(qm, 2, max_blocks, bs, n_block, table, free)
    want = assign_ref(table, free, n_block - 1, held_, new, bs, T, max_blocks, n_block)
    got = run_assign(qm, pool, held_, new, n_block - 1, T)
    assert got["status"][0] == want[0] == 0 and np.array_equal(pool.read()[0], want[1])
    for k, w in zip(("slot", "pos", "cu", "len"), want[2:6]):
        assert np.array_equal(got[k], w), k
    ln, nf, st = ints(qm, [9, 9]), ints(qm, [9]), ints(qm, [9])
    a, b, c = ints(qm, want[5]), ints(qm, [1, 1]), ints(qm, [want[6]])
    qm.kv_release_dev(pool.c, a.ptr, b.ptr, c.ptr, ln.ptr, nf.ptr, st.ptr)
    back = [x for i in range(2) for x in want[1][i, :-(-want[5][i] // bs)]]
    assert st.download(np.int32)[0] == 0 and nf.download(np.int32)[0] == n_block
    assert np.array_equal(pool.read()[1][want[6]:want[6] + len(back)], back)


@pytest.mark.parametrize("n_seq", [3, 256, 257, 600, 4096])
def test_assign_and_release_of_several_faults(qm, n_seq):
    """The status is the same whichever sequences have the faults: a length ahead of a row ahead of the
    list ahead of too few blocks."""
    bs, max_blocks, n_block, T = 16, 4, 12, 100
    pool = Pool(qm, n_seq, max_blocks, bs, n_block, np.full((n_seq, max_blocks), -1), np.arange(n_block))
    row, many_, neg = (70, 0), (0, 101), (0, -1)

    def assign(faults, top):
        held_, new = np.zeros(n_seq, int), np.zeros(n_seq, int)
        for at, (h, w) in faults.items():
            held_[at], new[at] = h, w
        return run_assign(qm, pool, held_, new, top, T)["status"][0]
    for i, j in ((0, 1), (1, 0), (0, n_seq - 1), (n_seq - 2, n_seq - 1), (n_seq - 1, n_seq - 2)):
        assert assign({i: row, j: many_}, 12) == 3 and assign({i: row, j: neg}, 12) == 3
        assert assign({i: row, j: (0, 30)}, 13) == 2 and assign({i: (0, 60), j: (0, 30)}, 13) == 4
        assert assign({i: (0, 60), j: (0, 30)}, 5) == 1 and assign({i: (0, 60), j: (0, 30)}, 6) == 0
        held_, ended = np.zeros(n_seq, int), np.zeros(n_seq, int)
        held_[[i, j]], ended[[i, j]] = (70, -1), 1
        ln, nf, st = ints(qm, held_), ints(qm, [9]), ints(qm, [9])
        a, b, c = ints(qm, held_), ints(qm, ended), ints(qm, [0])
        qm.kv_release_dev(pool.c, a.ptr, b.ptr, c.ptr, ln.ptr, nf.ptr, st.ptr)
        assert st.download(np.int32)[0] == 3


# ------------------------------------------------------------------------- far apart --

@pytest.mark.parametrize("layout", ["tokens", "heads"])
def test_strides_beyond_32_bits(qm, layout):
    """q, k, v and the results side by side in rows 2^31 values apart: by token, and by head."""
    t, D, S, gap = BF16, 64, (1 << 31) + 64, 512
    T, H = (3, 2) if layout == "tokens" else (40, 3)
    rows, inner = (T, H) if layout == "tokens" else (H, T)                # rows far apart, values within them
    r = rng_of(T, H, 97)
    a = {n: to_type(r.randn(T, H, D), t) for n in "qkv"}
    at = {n: i * inner * D for i, n in enumerate(("q", "k", "v", "rq", "rk", "op", "oc"))}
    buf = qm.DBuf(2 * ((rows - 1) * S + 7 * inner * D + gap))
    strides = (S, D) if layout == "tokens" else (D, S)
    view = lambda n: qm.heads((buf.ptr + 2 * at[n], H, *strides))  # noqa: E731
    near = lambda x: x if layout == "tokens" else x.transpose(1, 0, 2)  # noqa: E731

    def put(n, x):
        for i, row in enumerate(near(x)):
            buf.upload(np.ascontiguousarray(row), 2 * (i * S + at[n]))

    def get(n):
        got = np.stack([buf.download(np.uint16, inner * D, 2 * (i * S + at[n])) for i in range(rows)])
        return values(near(got.reshape(rows, inner, D)), t)
    for n in "qkv":
        put(n, a[n])
    pos, cu, slot = ints(qm, np.arange(T)), ints(qm, [0, T]), ints(qm, np.arange(T))
    both = lambda x, y: (qm.Heads * 2)(view(x)[0], view(y)[0])  # noqa: E731
    qm.rope_dev(qm.Rope.make(D, D, (32,), theta=1e4), pos.ptr, T, t, both("q", "k"), both("rq", "rk"))
    qf, kf, vf = (values(a[n], t) for n in "qkv")
    for n, x in (("rq", qf), ("rk", kf)):
        want = rope(x, np.arange(T)[None], D, (32,), False, False, 1e4)
        close(get(n), want, (HALF[t] + 2.0 ** -20) * np.abs(x).max() * 2)
    tq, tk = get("rq"), get("rk")
    qm.attn_prompt_dev(t, D, view("rq"), view("rk"), view("v"), view("op"), cu.ptr, 1, T, 0.125)
    want, mag, es = attention(tq, tk, vf, np.arange(T), 0.125)
    close(get("op"), want, 2 * HALF[t] * (mag + np.abs(want)) + 1e-4)
    cache = qm.DBuf(4 * H * 16 * (D + D // 8))
    c = qm.Kv4(cache.ptr, 4, 16, H, D)
    qm.kv4_append_dev(c, t, view("rk"), view("v"), slot.ptr, T)
    table, lens = ints(qm, [[0, 1, 2, 3]]), ints(qm, [T])
    kt = qm.KvTable(1, 4, 16, 4, table.ptr, None)
    qm.attn_kv4_dev(c, kt, t, view("rq"), view("oc"), cu.ptr, lens.ptr, T, 0.125)
    hk, hv = held(tk.astype(np.float32)), held(vf.astype(np.float32))
    want, mag, es = attention(tq, hk, hv, np.arange(T), 0.125)
    close(get("oc"), want, kv4_tol(t, D, T, want, mag, es))


@pytest.mark.parametrize("typ", ["f16", "f32"])
def test_attn_prompt_of_a_million_tokens(qm, typ):
    """4096 prompts of up to 500 tokens, the largest list of them."""
    t = TYPES[typ]
    r = rng_of(98)
    lens = r.randint(0, 500, 4096)
    T, D = int(lens.sum()), 64
    base = [to_type(r.randn(5000, 1, D), t) for _ in range(3)]
    pick = [r.randint(0, 5000, T) for _ in range(3)]
    q, k, v = (b[p] for b, p in zip(base, pick))
    views = [View(qm, x, t) for x in (q, k, v)]
    out = View(qm, np.zeros_like(q), t)
    cu = np.concatenate([[0], np.cumsum(lens)])
    qm.attn_prompt_dev(t, D, *[x.heads for x in views], out.heads, ints(qm, cu).ptr, 4096, T, 0.125)
    got = out.read()[0]
    for i in [0, 1, 63, 64, 65, 2047, 4000, 4094, 4095]:
        s = slice(cu[i], cu[i + 1])
        if lens[i]:
            want, mag, es = attention(*(values(x[s], t) for x in (q, k, v)), np.arange(lens[i]), 0.125)
            close(values(got[s], t), want, prompt_tol(t, D, int(lens[i]), want, mag, es), i)
