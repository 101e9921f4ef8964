"""The attention entries where forms, lengths and magnitudes meet: lengths that are
none, values far apart in size, infinite keys, the forms that only large calls take."""
import numpy as np
import pytest

from attn_fixtures import BF16, F16, F32, HALF, TYPES, View, attention, held, ints, rope, to_type, values
from test_gpu_attn import CacheCase, check_kv4, close, kv4_tol, kv_values, prompt_tol, rng_of, run_kv4, run_prompt
from test_gpu_attn_wide import kv4_bound, many, prompt_bound

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


# ------------------------------------------------------------------ sums of scores --

@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("typ", TYPES)
def test_attn_kv4_scores_that_nearly_cancel(qm, typ, D, rows):
    """Keys of whole numbers from -8 to 7, queries of 1 to 1 + 15 / 128: the sums of products of codes
    are hundreds to thousands, need up to 20 bits, and the minima take most of them off again.  A
    value of V for each token, so that a channel is one token's weight.

    The sums are exact in fp32.  A score of up to 256 log2(e) is rounded when scaled and when the
    maximum is taken off: 2 x 370 x 2^-24 of an exponent, numerator and sum each: under 1e-4 of a
    weight.  Weights to 2^-11 (fp32 calls 2^-21), and where codes are taken less 8, as much of 8.
    The largest weight enters the product as 2^6 at least (a step of 1), where fp16's smallest half
    step is 2^-25: 15 x 2^-31 of a value."""
    t = TYPES[typ]
    r = rng_of(D, rows, 5)
    L, H, KV = 60, 8, 2
    k = r.randint(-8, 8, (L, KV, D)).astype(np.float32)
    k[..., ::64], k[..., 1::64] = -8, 7
    v = np.zeros((L, KV, D), np.float32)
    v[np.arange(L), :, np.arange(L)] = 15
    q = to_type(1 + r.randint(0, 16, (rows, H, D)) / 128.0, t)
    case = CacheCase(qm, r, [L + rows - 1], KV, D, 16, [np.concatenate([k, np.repeat(k[:1], rows - 1, 0)])],
                     [np.concatenate([v, np.zeros((rows - 1, KV, D), np.float32)])])
    got = values(run_kv4(qm, case, q, [rows], t, scale=1.0, pad=0), t)[..., :L]
    want = attention(values(q, t), case.k[0], case.v[0], L - 1 + np.arange(rows), 1.0)[0][..., :L]
    part = 2.0 ** -21 if t == F32 else 2.0 ** -11
    close(got, want, (HALF[t] + part + 1e-4) * want + 8 * part * (t != BF16) + 2.0 ** -27 + 2.0 ** -25 * (t == F16))


@pytest.mark.parametrize("large", [0, 128, 4096])
@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("typ", TYPES)
def test_attn_kv4_scores_close_to_one_another(qm, typ, D, rows, large):
    """As above, with keys that hold the same numbers in another order; and with queries of 128 or
    4096 in every fourth channel, where all keys are 0, the others 1 to 1 + 15 / 16: products of up to
    2^15 beside such of 2^-4, all of whose sums are whole multiples of 2^-4 below 2^20, so exact in fp32.

    Where codes are taken less 8, what the other tokens leave of 8 is rounded by the sums too: up to
    130 tokens in 5 tiles, two products each, and 40 additions of minima, each to 2^-24 of 8."""
    t = TYPES[typ]
    r = rng_of(D, rows, 6)
    L, H, KV = 60, 8, 2
    one = r.randint(-8, 8, 64)
    one[:2] = -8, 7
    k = np.stack([np.concatenate([r.permutation(one) for _ in range(KV * D // 64)]).reshape(KV, D) for _ in range(L)]).astype(np.float32)
    v = np.zeros((L, KV, D), np.float32)
    v[np.arange(L), :, np.arange(L)] = 15
    q = 1 + r.randint(0, 16, (rows, H, D)) / (16.0 if large else 128.0)
    if large:
        k[..., 2::4], k[..., 0::64], k[..., 1::64], q[..., 2::4] = 0, -8, 7, large
    q = to_type(q, t)
    case = CacheCase(qm, r, [L + rows - 1], KV, D, 16, [np.concatenate([k, np.repeat(k[:1], rows - 1, 0)])],
                     [np.concatenate([v, np.zeros((rows - 1, KV, D), np.float32)])])
    got = values(run_kv4(qm, case, q, [rows], t, scale=1.0, pad=0), t)[..., :L]
    want = attention(values(q, t), case.k[0], case.v[0], L - 1 + np.arange(rows), 1.0)[0][..., :L]
    part = 2.0 ** -21 if t == F32 else 2.0 ** -11
    close(got, want, (HALF[t] + part + 1e-4) * want + 8 * (part + 52 * 2.0 ** -24) * (t != BF16) + 2.0 ** -27)


# ------------------------------------------------------ values far apart in size --

def one_far_key(r, L, KV, D, at, power, small, key=-120):
    """Normal keys and values (times `small`), but at token `at` a key of -120 in channel 0 and values
    2^power times as large.  For queries that hold 8 there."""
    k, v = r.randn(L, KV, D).astype(np.float32), (small * r.randn(L, KV, D)).astype(np.float32)
    k[:, :, 0] = 0
    k[at], k[at, :, 0] = 0, key
    v[at] = v[at] * np.float32(2.0 ** power)
    return k, v


def far_query(r, rows, H, D):
    q = r.randn(rows, H, D)
    q[..., 0] = 8
    return q


def norm_error(got, want):
    return np.linalg.norm(got - want) / np.linalg.norm(want)


@pytest.mark.parametrize("at", [0, 40, 290])
@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("typ", TYPES)
def test_attn_kv4_large_values_of_no_weight(qm, typ, D, rows, at):
    """A key of weight e^-40 and less whose values' step is 2^20 times the others': it has no part in
    the result, so the result is as exact as without it (the bound for normal inputs, of whose
    rounding terms the eight of a query's channel adds one of D as large as sqrt(D) others)."""
    t = TYPES[typ]
    r = rng_of(D, rows, at, 8)
    L, H, KV = 300 + rows, 4, 2
    k, v = one_far_key(r, L, KV, D, at, 20, 2.0 ** -8)
    case = CacheCase(qm, r, [L], KV, D, 16, [k], [v])
    q = to_type(far_query(r, rows, H, D), t)
    got = values(run_kv4(qm, case, q, [rows], t, pad=0), t)
    want = attention(values(q, t), case.k[0], case.v[0], L - rows + np.arange(rows), D ** -0.5)[0]
    assert norm_error(got, want) <= 2 * kv4_bound(t, D, L)


@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("typ", TYPES)
def test_attn_kv4_values_without_a_step(qm, typ, rows):
    """All values of a token alike (a step of 0), those of a few tokens not, and of one that nothing sees."""
    t = TYPES[typ]
    r = rng_of(rows, 81)
    L, H, KV, D = 400, 4, 2, 128
    k = r.randn(L, KV, D).astype(np.float32)
    v = np.repeat(r.randn(L, KV, 1), D, 2).astype(np.float32)
    q = to_type(r.randn(rows, H, D), t)
    for some in ([], [3], [200, 201], [399]):
        v2 = v.copy()
        v2[some] = 1000 * r.randn(len(some), KV, D)
        case = CacheCase(qm, r, [L], KV, D, 16, [k], [v2])
        got = values(run_kv4(qm, case, q, [rows], t, pad=0), t)
        want, mag, es = attention(values(q, t), case.k[0], case.v[0], L - rows + np.arange(rows), D ** -0.5)
        close(got, want, kv4_tol(t, D, L, want, 10 * mag, es), some)


@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("typ", TYPES)
def test_attn_kv4_a_nan_among_values(qm, typ, D, rows):
    """It takes its 64 channels, and no digit of the others."""
    t = TYPES[typ]
    r = rng_of(D, rows, 82)
    L, H, KV = 200 + rows, 4, 2
    k, v = (r.randn(L, KV, D).astype(np.float32) for _ in range(2))
    v[50, :, 70] = np.nan
    case = CacheCase(qm, r, [L], KV, D, 16, [k], [v])
    q = to_type(r.randn(rows, H, D), t)
    got = values(run_kv4(qm, case, q, [rows], t, pad=0), t)
    want = attention(values(q, t), case.k[0], case.v[0], L - rows + np.arange(rows), D ** -0.5)[0]
    gone = np.arange(D) // 64 == 1
    assert np.isnan(got[..., gone]).all() and np.isnan(want[..., gone]).all()
    assert norm_error(got[..., ~gone], want[..., ~gone]) <= kv4_bound(t, D, L)


PROMPT_FORMS = [(60, 4), (300, 4), (300, 0)]         # one launch; few workgroups; many (0: as many heads as it takes)


def prompt_error(qm, q, k, v, t, heads, but):
    """Norm-wise error of some of the heads of a prompt over one kv head, all rows but one."""
    T, H, D = q.shape
    got = values(run_prompt(qm, q, k, v, [T], t), t)[:, heads]
    want = attention(values(q, t)[:, heads], values(k, t), values(v, t), np.arange(T), D ** -0.5)[0]
    rows = np.arange(T) != but
    return norm_error(got[rows], want[rows])


@pytest.mark.parametrize("power", [12, 24, 60, 110])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T,H", PROMPT_FORMS)
@pytest.mark.parametrize("typ", TYPES)
def test_attn_prompt_large_values_of_no_weight(qm, typ, T, H, D, power):
    """As over the cache; the key is the second of the prompt or one of its last, so that rows meet it
    before, with and after the others."""
    t = TYPES[typ]
    if t == F16:
        power //= 10
    r = rng_of(D, T, power, 9)
    H = H or many(t, D)
    for at in (1, T - 20):
        # a weight of e^-60, or e^-120: 2^60 and 2^110 times that are nothing beside the others
        k, v = one_far_key(r, T, 1, D, at, power, 1.0, -7.5 * D ** 0.5 * (2 if power > 60 else 1))
        q = far_query(r, T, H, D)
        q[at, :, 0] = 0                              # in its own row it has weight: that one is large
        err = prompt_error(qm, *(to_type(x, t) for x in (q, k, v)), t, [0, H // 2, H - 1], at)
        assert err <= 2 * prompt_bound(t, D, T), at


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("typ", TYPES)
def test_attn_prompt_many_small_weights(qm, typ, D):
    """4095 keys of weights about e^-18 (2^-26) of the first one's, which has values of 0: together
    they are the result.  Each weight is held to the type's half step, or in fp16 to half its smallest
    step, 2^-25, of a largest weight of 2^7."""
    t = TYPES[typ]
    r = rng_of(D, 83)
    T, H = 4096, 2
    q, k, v = np.zeros((T, H, D)), 0.2 * r.randn(T, 1, D), r.randn(T, 1, D) + 2
    q[..., 0], k[:, 0, 0], v[0] = D ** 0.5, 0.5 * r.randn(T), 0
    k[0, 0, 0] = 18
    q, k, v = (to_type(x, t) for x in (q, k, v))
    got = values(run_prompt(qm, q, k, v, [T], t), t)
    rows = [0, 1, 1000, 2047, 3000, 4095]
    want, mag, es = attention(values(q, t)[rows], values(k, t), values(v, t), rows, D ** -0.5)
    e = es * (3 * 2.0 ** -22 * (t == F32) + (D + 16) * 2.0 ** -24)
    w = 3 * 2.0 ** -22 if t == F32 else HALF[t]
    tol = (2 * e + w + (T + 64) * 2.0 ** -24) * mag + HALF[t] * np.abs(want)
    close(got[rows], want, tol + (T * 2.0 ** -32 * 6 + 2.0 ** -25) * (t == F16) + 1e-30)


# -------------------------------------------------------------------- infinite keys --

def weigh64(q, k, v, scale):
    """One head of one prompt in 64 bits, infinite and NaN scores as they fall."""
    with np.errstate(all="ignore"):
        s = (q[:, None] * k[None]).sum(-1) * scale
        s[np.triu_indices(len(s), 1)] = -np.inf
        seen = np.tril(np.ones(s.shape, bool))
        p = np.where(seen, np.exp(s - np.where(seen, s, -np.inf).max(1, keepdims=True)), 0)
        return p @ v / p.sum(1, keepdims=True)


@pytest.mark.parametrize("scale", [0.125, -0.125, 0.0])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T,H", PROMPT_FORMS)
@pytest.mark.parametrize("typ", TYPES)
def test_attn_prompt_infinite_keys(qm, typ, T, H, D, scale):
    """A score of -inf is no weight, of +inf or NaN (infinities that meet, 0 times one) a row of NaN;
    a row that sees nothing else is NaN.  Rows that do not see the key are as they were."""
    t = TYPES[typ]
    r = rng_of(D, T, 84)
    H = H or many(t, D)
    heads = [0, H // 2, H - 1]
    q, k, v = r.randn(T, H, D), r.randn(T, 1, D), r.randn(T, 1, D)
    q[..., 3] = -np.abs(q[..., 3])
    q[30, :, 5], q[31, :, 3] = 0, 0
    clean = [to_type(x, t) for x in (q, k, v)]
    plain = values(run_prompt(qm, *clean, [T], t, scale=scale), t)[:, heads]
    qf, _, vf = (values(x, t) for x in clean)
    for places in ({(8, 3): np.inf}, {(0, 3): np.inf}, {(20, 5): -np.inf}, {(9, 3): np.inf, (9, 5): np.inf, (40, 3): np.inf},
                   {(12, 3): np.inf, (33, 3): np.inf, (T - 1, 3): np.inf}, {(T - 2, 7): np.nan}):
        k2 = k.copy()
        for (at, c), x in places.items():
            k2[at, 0, c] = x
        a = [clean[0], to_type(k2, t), clean[2]]
        got = values(run_prompt(qm, *a, [T], t, scale=scale), t)[:, heads]
        first = min(at for at, _ in places)
        assert np.array_equal(got[:first], plain[:first])
        kf = values(a[1], t)
        kz = np.where(np.isfinite(kf), kf, 0)
        for j, h in enumerate(heads):
            want = weigh64(qf[:, h], kf[:, 0], vf[:, 0], scale)
            _, mag, es = attention(qf[:, h:h + 1], kz, vf, np.arange(T), scale)
            nan = np.isnan(want)
            assert np.array_equal(np.isnan(got[:, j]), nan), (places, h)
            # a key without weight leaves the others the more: up to all of what the rows' first keys had
            tol = prompt_tol(t, D, T, want, 8 * mag[:, 0] + 8, es[:, 0])
            close(np.where(nan, 0, got[:, j]), np.where(nan, 0, want), np.where(nan, 1, tol), (places, h))


# ------------------------------------------------------------------------- angles --

def test_rope_near_half_turns(qm):
    """Angles close to odd and even multiples of pi, whose sines are 1e-5 to 1e-2: each comes out with
    the digits of fp32, as an angle formed in 64 bits has them (its frequency and product off by 2^-53
    each, pi by as much; sine and cosine by 2 of their own steps, the rest roundings)."""
    at = np.arange(1, 1 << 20)
    pos = at[np.abs(np.sin(at)) < 2e-3]
    T, D = len(pos), 64
    assert 355 in pos and T > 1000
    x = np.zeros((T, 1, D), np.float32)
    x[..., 0], x[1::2, :, 32] = 1, 1e-4
    xd, od = View(qm, x, F32), View(qm, np.zeros_like(x), F32)
    qm.rope_dev(qm.Rope.make(D, D, (32,), False, False, 1e4), ints(qm, pos).ptr, T, F32, xd.heads, od.heads)
    want = rope(x.astype(np.float64), pos[None], D, (32,), False, False, 1e4)
    got = od.read()[0].astype(np.float64)
    for c, other in ((0, 32), (32, 0)):
        a, b = np.abs(x[:, 0, c] * np.cos(pos)), np.abs(x[:, 0, other] * np.sin(pos))
        close(got[:, 0, c], want[:, 0, c], (a + b) * 5 * 2.0 ** -24 + 2.0 ** -51 * pos)


@pytest.mark.parametrize("T,H", PROMPT_FORMS)
@pytest.mark.parametrize("D", [64, 256])
def test_attn_prompt_huge_and_apart(qm, T, H, D):
    """Queries and keys of 1e38 in channels of their own: scores of 0, whose two powers of two together
    leave fp32's range."""
    r = rng_of(T, D, 85)
    H = H or many(F32, D)
    q, k, v = np.zeros((T, H, D), np.float32), np.zeros((T, 1, D), np.float32), r.randn(T, 1, D).astype(np.float32)
    q[..., ::2], k[..., 1::2] = 1e38, -1e38
    got = run_prompt(qm, q, k, v, [T], F32)[:, [0, H - 1]].astype(np.float64)
    want = np.cumsum(v[:, 0].astype(np.float64), 0) / np.arange(1, T + 1)[:, None]
    mag = np.cumsum(np.abs(v[:, 0]).astype(np.float64), 0) / np.arange(1, T + 1)[:, None]
    for h in range(2):
        close(got[:, h], want, (3 * 2.0 ** -22 + (T + 64) * 2.0 ** -24) * mag)


@pytest.mark.parametrize("sign,scale", [(1, 0.1), (-1, 0.1), (1, 4.0), (-1, 4.0)])
@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("typ", TYPES)
def test_attn_kv4_scores_beyond_their_own_units(qm, typ, D, rows, sign, scale):
    """Scores of 1e6 to 5e9, whose spacing in fp32 is up to 512: a row is the value of its largest key,
    which leads by more than the sums round (257 x 2^-24 of 6 times a score) and the weights keep."""
    t = TYPES[typ]
    r = rng_of(D, rows, 86)
    L, H, KV = 260 + rows, 4, 2
    k, v = r.randn(L, KV, D), r.randn(L, KV, D)
    k[..., 0] = sign * (3000 + 60000.0 * r.permutation(L)[:, None] / L)
    q = r.randn(rows, H, D)
    q[..., 0] = 20000 + 1000 * r.rand(rows, H)
    q = to_type(q, t)
    case = CacheCase(qm, r, [L], KV, D, 16, [k.astype(np.float32)], [v.astype(np.float32)])
    got = values(run_kv4(qm, case, q, [rows], t, scale=scale, pad=0), t)
    qf, want = values(q, t), np.zeros((rows, H, D))
    for j in range(rows):
        n = L - rows + j + 1
        for h in range(H):
            s = case.k[0][:n, h // 2] @ qf[j, h] * scale
            two = np.partition(s, -2)[-2:]
            assert two[1] - two[0] > 257 * 6 * 2.0 ** -24 * np.abs(s).max() + 100
            want[j, h] = case.v[0][s.argmax(), h // 2]
    part = 2.0 ** -21 if t == F32 else 2.0 ** -10
    close(got, want, HALF[t] * np.abs(want) + 16 * part)


@pytest.mark.parametrize("sign,scale", [(1, 0.1), (-1, 0.1), (1, 4.0), (-1, 4.0)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T,H", PROMPT_FORMS)
@pytest.mark.parametrize("typ", TYPES)
def test_attn_prompt_scores_beyond_their_own_units(qm, typ, T, H, D, sign, scale):
    """As over the cache: every row is the value of the largest key that it sees, or of several whose
    scores are within what the sums round."""
    t = TYPES[typ]
    r = rng_of(D, T, 87)
    H = H or many(t, D)
    q, k, v = r.randn(T, H, D), r.randn(T, 1, D), r.randn(T, 1, D)
    k[..., 0] = sign * (3000 + 60000.0 * r.permutation(T)[:, None] / T)
    q[..., 0] = 20000 + 1000 * r.rand(T, H)
    q, k, v = (to_type(x, t) for x in (q, k, v))
    got = values(run_prompt(qm, q, k, v, [T], t, scale=scale), t)
    qf, kf, vf = values(q, t), values(k, t)[:, 0], values(v, t)[:, 0]
    sure = 0
    for h in (0, H - 1):
        s = qf[:, h] @ kf.T * scale
        for j in range(T):
            a = s[j, :j + 1]
            near = a > a.max() - D * 6 * 2.0 ** -24 * np.abs(a).max() - 200
            if near.sum() == 1:
                sure += 1
                close(got[j, h], vf[a.argmax()], 2 * HALF[t] * np.abs(vf[a.argmax()]) + 2.0 ** -20, (j, h))
            else:
                assert (got[j, h] <= vf[:j + 1][near].max(0) + 0.1).all() and (got[j, h] >= vf[:j + 1][near].min(0) - 0.1).all(), (j, h)
    assert sure


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T,H", PROMPT_FORMS)
@pytest.mark.parametrize("typ", TYPES)
def test_attn_prompt_huge_keys_that_are_seen(qm, typ, T, H, D):
    """Finite keys near the type's largest value: a row whose score there is positive is that key's
    value, for the others the key has no weight."""
    t = TYPES[typ]
    r = rng_of(D, T, 88)
    H = H or many(t, D)
    q, k, v = r.randn(T, H, D), r.randn(T, 1, D), r.randn(T, 1, D)
    q[..., 3] = np.where(q[..., 3] < 0, -1, 1) * (0.5 + r.rand(T, H))
    big = 6e4 if t == F16 else 1e38
    k[20, 0, 3], k[41, 0, 3], k[T - 3, 0, 3] = big, big * 0.75, -big
    q, k, v = (to_type(x, t) for x in (q, k, v))
    got = values(run_prompt(qm, q, k, v, [T], t, scale=0.125), t)
    calm = values(k, t)
    calm = np.where(np.abs(calm) > 100, 0, calm)
    for h in (0, H // 2, H - 1):
        want = weigh64(values(q, t)[:, h], values(k, t)[:, 0], values(v, t)[:, 0], 0.125)
        _, mag, es = attention(values(q, t)[:, h:h + 1], calm, values(v, t), np.arange(T), 0.125)
        close(got[:, h], want, prompt_tol(t, D, T, want, 8 * mag[:, 0] + 8, es[:, 0]), h)


@pytest.mark.parametrize("typ", ["f32", "bf16"])
@pytest.mark.parametrize("T,H", PROMPT_FORMS)
def test_attn_prompt_lowest_scores(qm, typ, T, H):
    """All scores -2.2e38, times log2(e) near fp32's lowest value: they are equal, so a row is a mean."""
    t = TYPES[typ]
    r = rng_of(T, 89)
    D, H = 64, H or many(t, 64)
    q, k, v = np.zeros((T, H, D)), np.zeros((T, 1, D)), r.randn(T, 1, D)
    q[..., 0], k[..., 0] = 1, -2.2e38
    q, k, v = (to_type(x, t) for x in (q, k, v))
    got = values(run_prompt(qm, q, k, v, [T], t, scale=1.0), t)
    vf = values(v, t)[:, 0]
    n = np.arange(1, T + 1)[:, None]
    want, mag = np.cumsum(vf, 0) / n, np.cumsum(np.abs(vf), 0) / n
    for h in (0, H - 1):
        close(got[:, h], want, (3 * 2.0 ** -22 + (T + 64) * 2.0 ** -24) * mag + HALF[t] * np.abs(want))


@pytest.mark.parametrize("size", ["largest", "small"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T,H", PROMPT_FORMS + [(2500, 4)])
@pytest.mark.parametrize("typ", TYPES)
def test_attn_prompt_values_of_any_size(qm, typ, T, H, D, size):
    """Values near the type's largest, whose sums would leave fp32's range, and small ones: their means
    are as exact as those of others."""
    t = TYPES[typ]
    r = rng_of(T, D, 90)
    H = H or many(t, D)
    big = {F32: 3e38, BF16: 3e38, F16: 6e4}[t] if size == "largest" else {F32: 1e-25, BF16: 1e-25, F16: 1.0}[t]
    q, k, v = (to_type(x, t) for x in (r.randn(T, H, D), r.randn(T, 1, D), big * (0.5 + 0.5 * r.rand(T, 1, D))))
    got = values(run_prompt(qm, q, k, v, [T], t), t)
    rows = np.unique(np.concatenate([np.arange(0, T, 61), [1, 31, 32, T - 1]]))
    for h in (0, H - 1):
        want, mag, es = attention(values(q, t)[rows, h:h + 1], values(k, t), values(v, t), rows, D ** -0.5)
        assert norm_error(got[rows, h] / big, want[:, 0] / big) <= prompt_bound(t, D, T)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T,H", PROMPT_FORMS + [(2500, 4)])
@pytest.mark.parametrize("typ", ["f16", "bf16"])
def test_attn_prompt_is_a_mean_of_values(qm, typ, T, H, D):
    """All values the type's largest: so is every result, whatever the weights' rounding; and a row of
    one or two keys, whose weights' rounding takes no part in it or little, is off by its own."""
    t = TYPES[typ]
    r = rng_of(T, D, 91)
    H = H or many(t, D)
    top = np.float32(65504) if t == F16 else np.array([0x7F7F0000], np.uint32).view(np.float32)[0]
    q, k = to_type(r.randn(T, H, D), t), to_type(r.randn(T, 1, D), t)
    got = values(run_prompt(qm, q, k, to_type(np.full((T, 1, D), top), t), [T], t), t)
    assert (got == top).all()
    v = to_type(r.randn(T, 1, D), t)
    got = values(run_prompt(qm, q, k, v, [T], t), t)
    assert np.array_equal(got[0], np.repeat(values(v, t)[0], H, 0))
