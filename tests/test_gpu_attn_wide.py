"""More of the attention entries: errors as a whole against 64 bits, the kernels
that large calls take, calls one behind another, a cache beyond 4 GiB."""
import numpy as np
import pytest

from attn_fixtures import BF16, F16, F32, TYPES, View, attention, held, ints, quantise, to_type, values
from test_gpu_attn import (CacheCase, check_kv4, check_prompt, close, kv4_tol, kv_values, prompt_tol, rng_of, run_kv4,
                           run_prompt)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------- errors as a whole --
#
# 2-norm of the error over 2-norm of the result.  Normal q, k and v, scale D^-0.5.
#
# fp32: a score is D products of rms 1, summed in fp32: every addition rounds by
# at most 2^-24 of the sum so far (rms up to sqrt(D)), in either direction, so
# D^0.5 D^0.5 2^-24, which the scale makes D^0.5 2^-24; codes and minimum apart
# are two such sums.  That is a weight's relative error; the operands' parts leave
# 2^-22 of q and of the weight (prompts: of k and v too).  L weights are summed 16
# at a time: (L / 16)^0.5 2^-24 of the result.
#
# 16 bits: rounding a value of p bits is off by 2^(1 - p) / 12^0.5 of the power of
# two below it, 2^(1 - p) / 24^0.5 of the value in the mean over a factor of two
# (fp16 2.0e-4, bf16 1.6e-3).  The result is rounded to the type, the weights to
# the type (prompts) or to fp16 (cache), each independently of the others and of
# the v it multiplies, so that their errors add up as the weights themselves do:
# as much again, times the operand's rms over v's.  That is 1.03 for code - 8 of
# 64 normal values (rms 3.3 steps of a spread of 4.7 / 15) and 2.8 for the code
# itself.  bf16 decode on subnormal codes sums 10 of 24 bits short: 2^-14 of up to
# ten times the result.  A tenth more for these being samples.

def kv4_bound(t, D, L):
    if t == F32:
        return 2 * (D ** 0.5 + (L / 16) ** 0.5) * 2.0 ** -24 + 2 * 2.0 ** -22
    f16, bf16 = 2.0 ** -10 / 24 ** 0.5, 2.0 ** -7 / 24 ** 0.5
    if t == F16:
        return 1.1 * f16 * (1 + 1.03 ** 2) ** 0.5
    return 1.1 * (bf16 ** 2 + (2.8 * f16) ** 2 + (10 * 2.0 ** -14) ** 2) ** 0.5


def prompt_bound(t, D, L):
    if t == F32:
        return (D ** 0.5 + (L / 16) ** 0.5) * 2.0 ** -24 + 4 * 2.0 ** -22
    return 1.1 * 2 ** 0.5 * (2.0 ** -10 if t == F16 else 2.0 ** -7) / 24 ** 0.5


def error(got, want):
    return np.linalg.norm(got - want) / np.linalg.norm(want)


@pytest.mark.parametrize("rows", [1, 60, 70])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("typ", TYPES)
def test_attn_kv4_error(qm, typ, D, rows):
    """Both kernels: few rows to a sequence and many."""
    t = TYPES[typ]
    r = rng_of(D, rows, 77)
    lens, H, KV = ([700, 300, 512, 131], 8, 2) if rows == 1 else ([700], 8, 2)
    k, v = ([r.randn(n, KV, D).astype(np.float32) for n in lens] for _ in range(2))
    case = CacheCase(qm, r, lens, KV, D, 32, k, v)
    ask = [rows] * len(lens)
    q = to_type(r.randn(sum(ask), H, D), t)
    got = values(run_kv4(qm, case, q, ask, t, pad=0), t)
    want = np.concatenate([attention(values(q[i * rows:(i + 1) * rows], t), case.k[i], case.v[i], n - rows + np.arange(rows),
                                     D ** -0.5)[0] for i, n in enumerate(lens)])
    assert error(got, want) <= kv4_bound(t, D, max(lens))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("typ", TYPES)
def test_attn_prompt_error(qm, typ, D):
    t = TYPES[typ]
    r = rng_of(D, 78)
    lens = [400, 120]
    q, k, v = (to_type(r.randn(520, n, D), t) for n in (2, 1, 1))
    got = values(run_prompt(qm, q, k, v, lens, t), t)
    qf, kf, vf = (values(x, t) for x in (q, k, v))
    want = np.concatenate([attention(qf[a:b], kf[a:b], vf[a:b], np.arange(b - a), D ** -0.5)[0] for a, b in ((0, 400), (400, 520))])
    assert error(got, want) <= prompt_bound(t, D, 400)


# --------------------------------------------------- prompts of many workgroups --

def many(t, D):
    """Query heads for which a few hundred tokens are a large call."""
    return 32 if t == F32 and D == 256 else 120


def subset(a, H, KV):
    heads = np.unique([0, H // 2 - 1, H - 1])
    return heads, heads // (H // KV)


@pytest.mark.parametrize("layout", ["packed", "odd"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("typ", TYPES)
def test_attn_prompt_large(qm, typ, D, layout):
    """Ragged lengths, empty prompts and rows behind the last one."""
    t = TYPES[typ]
    H, KV, lens, pad = many(t, D), 8, [129, 31, 1, 64, 0, 200, 32], 3
    r = rng_of(D, 5, 12)
    T = sum(lens) + pad
    q, k, v = to_type(r.randn(T, H, D), t), to_type(kv_values(r, (T, KV, D)), t), to_type(r.randn(T, KV, D), t)
    got = run_prompt(qm, q, k, v, lens, t, layout)
    qh, kh = subset(q, H, KV)
    at = 0
    for n in lens:
        s = slice(at, at + n)
        at += n
        for a, b in zip(qh, kh):
            want, mag, es = attention(*(values(x[s, c:c + 1], t) for x, c in ((q, a), (k, b), (v, b))), np.arange(n), D ** -0.5)
            if n:
                close(values(got[s, a:a + 1], t), want, prompt_tol(t, D, n, want, mag, es), (n, a))


@pytest.mark.parametrize("few", [False, True])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("typ", TYPES)
def test_attn_prompt_large_is_not_reached_by_what_it_does_not_see(qm, typ, D, few):
    """With many query heads, and with so few that a workgroup takes fewer queries."""
    t = TYPES[typ]
    H, KV, lens, T, at = 4 if few else many(t, D), 4, [150, 0, 40, 140, 1], 335, 70
    r = rng_of(D, 41)
    q, k, v = r.randn(T, H, D), kv_values(r, (T, KV, D)), r.randn(T, KV, D)
    want = values(run_prompt(qm, *(to_type(x, t) for x in (q, k, v)), lens, t), t)
    for bad in (np.nan, -np.inf, {F32: 3e38, BF16: 3e38, F16: 65504.0}[t]):
        kb, vb = k.copy(), v.copy()
        kb[at, :, 3], kb[331:] = bad, bad
        vb[at, :, 7], vb[331:] = bad, bad
        got = values(run_prompt(qm, *(to_type(x, t) for x in (q, kb, vb)), lens, t), t)
        seen = (np.arange(T) >= at) & (np.arange(T) < 150)
        live = ~seen & (np.arange(T) < 331)
        assert np.array_equal(got[live], want[live]), bad
        if not np.isfinite(bad):
            assert not np.isfinite(got[seen]).all()


@pytest.mark.parametrize("n,H", [(130, 600), (300, 2)])
@pytest.mark.parametrize("typ", TYPES)
def test_attn_prompt_large_infinite_values(qm, typ, n, H):
    """V's infinities keep their sign."""
    t = TYPES[typ]
    KV, D = 1, 64
    r = rng_of(9, 9)
    q, k, v = 0.1 * r.randn(n, H, D), 0.1 * r.randn(n, KV, D), r.randn(n, KV, D)
    v[65, 0, 2], v[100, 0, 2], v[70, 0, 63] = -np.inf, np.inf, np.inf
    got = values(run_prompt(qm, *(to_type(x, t) for x in (q, k, v)), [n], t), t)
    assert np.isfinite(got[:65]).all() and np.isneginf(got[65:100, :, 2]).all() and np.isnan(got[100:, :, 2]).all()
    assert np.isposinf(got[70:, :, 63]).all()
    got[65:, :, [2, 63]] = 0
    assert np.isfinite(got).all()


@pytest.mark.parametrize("cu", [[0, 130, 3], [-5, 2, 4], [0, 2, 1 << 30], [130, 0, 130], [0, 1 << 30, 1 << 30]])
def test_attn_prompt_large_bad_lengths(qm, cu):
    """Lengths that are none write no row outside the output (the results are not defined)."""
    r = rng_of(8, 3)
    for t, H in ((F32, 400), (BF16, 400)):
        q, k, v = (View(qm, to_type(r.randn(130, n, 64), t), t, "gap") for n in (H, 2, 2))
        out = View(qm, to_type(np.zeros((130, H, 64)), t), t, "gap", fill=3)
        qm.attn_prompt_dev(t, 64, q.heads, k.heads, v.heads, out.heads, ints(qm, cu).ptr, 2, 130, 0.125)
        assert out.read()[1]


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("n_seq,T,D", [(700, 40, 64), (4096, 300, 128)])
def test_attn_prompt_mostly_empty(qm, typ, n_seq, T, D):
    """Far more prompts than tokens: all but a few are empty."""
    t = TYPES[typ]
    r = rng_of(n_seq, T)
    lens = np.zeros(n_seq, int)
    lens[r.choice(n_seq, 7, replace=False)] = np.diff(np.concatenate([[0], np.sort(r.choice(np.arange(1, T), 6, replace=False)), [T]]))
    q, k, v = (to_type(r.randn(T, n, D), t) for n in (4, 2, 2))
    check_prompt(q, k, v, lens, t, run_prompt(qm, q, k, v, lens, t))


# ------------------------------------------------------- the cache, many rows --

@pytest.mark.parametrize("typ", TYPES)
def test_attn_kv4_many_rows_do_not_see_later_tokens(qm, typ):
    t = TYPES[typ]
    L, n, H, KV, D, bs = 330, 90, 8, 2, 128, 16
    r = rng_of(70, 8)
    k, v = kv_values(r, (L, KV, D)).astype(np.float32), r.randn(L, KV, D).astype(np.float32)
    q = to_type(r.randn(n, H, D), t)
    want = values(run_kv4(qm, CacheCase(qm, r, [L], KV, D, bs, [k], [v]), q, [n], t, pad=0), t)
    for bad in (np.nan, np.inf, 65000.0):
        k2, v2 = k.copy(), v.copy()
        k2[L - 30:, :, 5], v2[L - 30:, :, 70] = bad, bad
        dirty = CacheCase(qm, r, [L], KV, D, bs, [k2], [v2])
        got = values(run_kv4(qm, dirty, q, [n], t, pad=0), t)
        close(got[:n - 30], want[:n - 30], 2 * kv4_tol(t, D, L, want[:n - 30], 3.0, 20.0), bad)
        if bad != 65000.0:
            assert not np.isfinite(got[n - 30:]).all()


@pytest.mark.parametrize("D,layout", [(64, "odd"), (128, "packed"), (256, "gap")])
@pytest.mark.parametrize("typ", TYPES)
def test_attn_kv4_many_rows(qm, typ, D, layout):
    """Ragged lengths, more rows than tokens, sequences that ask nothing or have nothing."""
    t = TYPES[typ]
    r = rng_of(D, 31, 7)
    lens, ask = [300, 40, 0, 500, 33, 64], [290, 60, 3, 129, 0, 64]
    case = CacheCase(qm, r, lens, 2, D, 16)
    q = to_type(r.randn(sum(ask) + 2, 8, D), t)
    check_kv4(case, q, ask, t, run_kv4(qm, case, q, ask, t, layout))


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("rows", [1, 80])
def test_attn_kv4_bad_pages_anywhere(qm, typ, rows):
    """Pages that are not there, whole chunks of them, in a sequence that is split."""
    t = TYPES[typ]
    L, H, KV, D, bs = 1000, 8, 2, 64, 16
    r = rng_of(rows, 10)
    case = CacheCase(qm, r, [L], KV, D, bs)
    q = to_type(r.randn(rows, H, D), t)
    for columns, bad in (([0, 1, 30, 62], -1), (range(8, 40), case.n_block), (range(1, 63), 1 << 30)):
        table, gone = case.table.copy(), np.zeros(L, bool)
        for c in columns:
            table[0, c] = bad
            gone[c * bs:(c + 1) * bs] = True
        case.table_dev.upload(table.astype(np.int32))
        got = values(run_kv4(qm, case, q, [rows], t, pad=0), t)
        there = np.flatnonzero(~gone)
        last = np.searchsorted(there, L - rows + np.arange(rows), side="right") - 1
        want, mag, es = attention(values(q, t), case.k[0][there], case.v[0][there], last, D ** -0.5)
        close(got, want, kv4_tol(t, D, L, want, mag, es), (columns, bad))


def test_attn_kv4_many_sequences_split(qm):
    """More joined rows than a workgroup each for: twenty sequences of several parts."""
    r = rng_of(20, 20)
    lens = [900 + 40 * i for i in range(20)]
    for t in (F32, BF16):
        case = CacheCase(qm, r, lens, 2, 128, 64)
        q = to_type(r.randn(22, 16, 128), t)
        check_kv4(case, q, [1] * 20, t, run_kv4(qm, case, q, [1] * 20, t))


# ------------------------------------------------------ scales and odd queries --

@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
@pytest.mark.parametrize("typ", TYPES)
def test_scales(qm, typ, scale):
    """No scale (the mean of v), one that turns the order round, one that leaves a single token."""
    t = TYPES[typ]
    r = rng_of(int(10 * abs(scale)), 6)
    D, H, KV, L = 64, 4, 2, 200
    case = CacheCase(qm, r, [L], KV, D, 16)
    for rows in (1, 50, 150):
        q = to_type(r.randn(rows, H, D), t)
        check_kv4(case, q, [rows], t, run_kv4(qm, case, q, [rows], t, scale=scale, pad=0), scale)
    q, k, v = (to_type(r.randn(L, n, D), t) for n in (H, KV, KV))
    check_prompt(q, k, v, [L], t, run_prompt(qm, q, k, v, [L], t, scale=scale), scale)


@pytest.mark.parametrize("typ", TYPES)
def test_a_row_of_nan_stays_alone(qm, typ):
    """NaN, infinite and zero queries: their rows, and no other."""
    t = TYPES[typ]
    r = rng_of(61)
    D, H, KV, L = 128, 8, 2, 180
    k, v = (r.randn(L, KV, D).astype(np.float32) for _ in range(2))
    case = CacheCase(qm, r, [L], KV, D, 16, [k], [v])
    for rows in (3, 60, 90, L):                      # the last: a prompt
        q = r.randn(rows, H, D)
        run = ((lambda x: run_prompt(qm, x, to_type(k, t), to_type(v, t), [L], t)) if rows == L else
               (lambda x: run_kv4(qm, case, x, [rows], t, pad=0)))
        want = values(run(to_type(q, t)), t)
        q[0, 3, 5], q[1, 2, 7], q[2, 4] = np.nan, np.inf, 0
        got = values(run(to_type(q, t)), t)
        assert np.isnan(got[0, 3]).all() and not np.isfinite(got[1, 2]).all() and np.isfinite(got[2, 4]).all()
        for i, h in ((0, 3), (1, 2), (2, 4)):
            got[i, h] = want[i, h] = 0
        assert np.array_equal(got, want), rows


# ------------------------------------------------------------------- the cache --

@pytest.mark.parametrize("typ", TYPES)
def test_steps_half_way(qm, typ):
    """A spread of 15 times 4093: a step between two of fp16's, where quotient and product part."""
    t = TYPES[typ]
    D, bs, n = 128, 16, 9
    r = rng_of(4, 4)
    x = r.randint(45, 60000, (n, 1, D)) // 256 * 256 + 45.0
    x[:, :, ::64], x[:, :, 63::64] = 45.0, 61440.0
    x *= 2.0 ** -np.arange(n)[:, None, None]
    x = to_type(x, t)
    _, d, _ = quantise(values(x, t).astype(np.float32))
    assert (d[:, 0, 0].astype(np.float64) == 4094 * 2.0 ** -np.arange(n)).all()
    cache = qm.DBuf(bs * (D + D // 8))
    c = qm.Kv4(cache.ptr, 1, bs, 1, D)
    view, sl = View(qm, x, t), ints(qm, np.arange(n))
    qm.kv4_append_dev(c, t, view.heads, view.heads, sl.ptr, n)
    ko, vo = qm.DBuf(4 * n * D), qm.DBuf(4 * n * D)
    qm.kv4_read_dev(c, sl.ptr, n, ko.ptr, vo.ptr)
    want = held(values(x, t).astype(np.float32))
    for o in (ko, vo):
        assert np.array_equal(o.download(np.float32).reshape(n, 1, D).astype(np.float64), want)


def test_cache_beyond_4_gib(qm):
    """Blocks whose bytes lie past 32-bit offsets, and slots near the largest block."""
    KV, D, bs = 8, 256, 256
    n_block = (1 << 32) // (KV * bs * (D + D // 8)) + 40
    cache = qm.DBuf(n_block * KV * bs * (D + D // 8))
    c = qm.Kv4(cache.ptr, n_block, bs, KV, D)
    r = rng_of(3, 33)
    lens, L = [300, 40], 340
    pages = [[n_block - 1, n_block - 20], [n_block - 3, 0]]
    seq = np.repeat([0, 1], lens)
    tok = np.concatenate([np.arange(n) for n in lens])
    slot = np.array(pages)[seq, tok // bs] * bs + tok % bs
    k, v = kv_values(r, (L, KV, D)).astype(np.float32), r.randn(L, KV, D).astype(np.float32)
    kd, vd, sl = View(qm, k, F32), View(qm, v, F32), ints(qm, slot)
    qm.kv4_append_dev(c, F32, kd.heads, vd.heads, sl.ptr, L)
    ko, vo = qm.DBuf(4 * L * KV * D), qm.DBuf(4 * L * KV * D)
    qm.kv4_read_dev(c, sl.ptr, L, ko.ptr, vo.ptr)
    hk, hv = held(k), held(v)
    assert np.array_equal(ko.download(np.float32).reshape(k.shape), hk) and np.array_equal(vo.download(np.float32).reshape(v.shape), hv)
    table, len_d = ints(qm, pages), ints(qm, lens)
    t = qm.KvTable(2, 2, bs, n_block, table.ptr, None)
    for ask in ([1, 1], [70, 40], [300, 40]):
        n = sum(ask)
        q = r.randn(n, 16, D).astype(np.float32)
        qd, od = View(qm, q, F32), View(qm, np.zeros_like(q), F32)
        cu = ints(qm, np.cumsum([0] + ask))
        qm.attn_kv4_dev(c, t, F32, qd.heads, od.heads, cu.ptr, len_d.ptr, n, D ** -0.5)
        got, at = od.read()[0], 0
        for i, (m, s) in enumerate(zip(ask, (slice(0, 300), slice(300, 340)))):
            want, mag, es = attention(q[at:at + m].astype(np.float64), hk[s], hv[s], lens[i] - m + np.arange(m), D ** -0.5)
            close(got[at:at + m], want, kv4_tol(F32, D, lens[i], want, mag, es), (ask, i))
            at += m


# ------------------------------------------------------------------- together --

def test_calls_one_behind_another(qm):
    """Calls that share the workspace, queued without a wait between them: each has the result it
    has alone, and the profile counts them."""
    r = rng_of(14)
    D, KV, H = 128, 2, 8
    case = CacheCase(qm, r, [1500, 200, 900], KV, D, 32)
    len_d = ints(qm, case.lens)
    jobs = []
    for t, ask in ((F32, [1, 1, 1]), (BF16, [1, 0, 1]), (F32, [100, 60, 9]), (F16, [300, 1, 1])):
        n = sum(ask)
        q = View(qm, to_type(r.randn(n, H, D), t), t)
        o = View(qm, to_type(np.zeros((n, H, D)), t), t)
        cu = ints(qm, np.cumsum([0] + ask))
        jobs.append((o, (q, cu), lambda t=t, q=q, o=o, cu=cu, n=n: qm.attn_kv4_dev(
            case.c, case.t, t, q.heads, o.heads, cu.ptr, len_d.ptr, n, D ** -0.5)))
    for t, T in ((F32, 500), (BF16, 90)):
        x = [View(qm, to_type(r.randn(T, n, D), t), t) for n in (H, KV, KV)]
        o = View(qm, to_type(np.zeros((T, H, D)), t), t)
        cu = ints(qm, [0, T // 3, T])
        jobs.append((o, (x, cu), lambda t=t, T=T, x=x, o=o, cu=cu: qm.attn_prompt_dev(
            t, D, *[y.heads for y in x], o.heads, cu.ptr, 2, T, D ** -0.5)))
    alone = []
    for o, _, job in jobs:
        job()
        alone.append(o.read()[0].copy())
        o.buf.upload(o.host)
    order = list(range(len(jobs))) * 3
    r.shuffle(order)
    qm.prof_enable(True)
    try:
        for i in order:
            jobs[i][2]()
        assert qm.prof_read("attn")[0] == len(order)
    finally:
        qm.prof_enable(False)
    for (o, _, _), want in zip(jobs, alone):
        assert np.array_equal(o.read()[0].view(np.uint8), want.view(np.uint8))
