"""Log probabilities, entropy and the most likely tokens (qmag_logprobs_dev) against their
definitions in 64 bits."""
import numpy as np
import pytest

from attn_fixtures import BF16, F16, F32, TYPES, ints, to_type, values
from recurrent_fixtures import rng_of

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


def run(qm, x, t, token, k, stride=None, skip=()):
    """x [T][V] stored values; rows `stride` apart, junk between them."""
    T, V = x.shape
    stride = stride or V
    buf = np.full((max(T, 1), stride), to_type(np.float32(1e9 if t != F16 else 6e4), t))
    buf[:T, :V] = x
    xb, tb = qm.DBuf.from_array(buf), ints(qm, token)
    ob = {n: qm.DBuf.from_array(np.full(max(1, T * m) + 3, 77, dt)) for n, m, dt in
          (("logprob", 1, np.float32), ("entropy", 1, np.float32), ("id", k, np.int32), ("val", k, np.float32))}
    p = {n: None if n in skip else b.ptr for n, b in ob.items()}
    qm.logprobs_dev(V, t, xb.ptr, stride, None if "logprob" in skip else tb.ptr, T, k, p["logprob"], p["entropy"], p["id"], p["val"])
    got = {n: b.download(np.int32 if n == "id" else np.float32) for n, b in ob.items()}
    for n, m in (("logprob", 1), ("entropy", 1), ("id", k), ("val", k)):
        assert (got[n][T * m if n not in skip else 0:] == 77).all()
    return got["logprob"][:T], got["entropy"][:T], got["id"][:T * k].reshape(T, k), got["val"][:T * k].reshape(T, k)


def order(x):
    """Places by value, the lowest first among equal ones (-0 is +0), NaN last."""
    return np.argsort(np.where(np.isnan(x), np.inf, -(x + 0.0)) if not np.isnan(x).any() else
                      np.where(np.isnan(x), np.float64(2), -np.arctan(x.astype(np.float64))), kind="stable")


def check(qm, x, t, token, k, stride=None, skip=()):
    T, V = x.shape
    lp, ent, ids, val = run(qm, x, t, token, k, stride, skip)
    for i in range(T):
        v = values(x[i], t)
        m = v.max()
        d = v - m
        e = np.exp(d)
        Z = e.sum()
        some = e > 0
        mean, square = (e[some] * -d[some]).sum() / Z, (e[some] * d[some] ** 2).sum() / Z
        # e^d: its argument and the difference rounded (3 |d| 2^-24 of it), the function itself 2; groups of eight
        # added without loss but for a step, then at most some twenty joins of lanes, waves and parts, two roundings each
        off = (64 + 4 * mean) * EPS
        if "logprob" not in skip:
            tok = token[i]
            want = d[tok] - np.log(Z) if 0 <= tok < V else 0.0
            tol = off + EPS * (2 * abs(want) + 2 * abs(np.log(Z)) + 1e-30) if 0 <= tok < V else 0.0
            assert lp[i] == want or abs(lp[i] - want) <= tol, (i, lp[i], want, tol)
        if "entropy" not in skip:
            want = np.log(Z) + mean
            tol = off * (1 + mean) + 4 * EPS * (square + abs(np.log(Z)) + mean)
            assert abs(ent[i] - want) <= tol, (i, ent[i], want, tol)
        want = order(v)[:k]
        assert np.array_equal(ids[i], want), (i, ids[i], want)
        w = d[want] - np.log(Z)
        with np.errstate(invalid="ignore"):
            assert ((val[i] == w) | (np.abs(val[i] - w) <= off + EPS * (2 * np.abs(w) + 2 * abs(np.log(Z))))).all(), (i, val[i], w)


def logits(r, T, V, t, peaks=3):
    x = 2.5 * r.randn(T, V)
    x[np.arange(T)[:, None], r.randint(0, V, (T, peaks))] += r.uniform(2, 16, (T, peaks))
    return to_type(x, t)


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 511, 513, 2047, 2049, 4099, 32003])
@pytest.mark.parametrize("T", [1, 5])
def test_logprobs_sizes(qm, typ, V, T):
    r = rng_of(V, T)
    check(qm, logits(r, T, V, TYPES[typ]), TYPES[typ], r.randint(0, V, T), min(V, 20), stride=V + T - 1)


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("k", [0, 1, 2, 20, 63, 64])
def test_logprobs_alternatives(qm, typ, k):
    r = rng_of(k)
    for T, V in ((3, 9001), (2, 64)):
        check(qm, logits(r, T, V, TYPES[typ]), TYPES[typ], r.randint(0, V, T), k)


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("T,V,k", [(1500, 70, 5), (1024, 2500, 3), (1100, 700, 64), (600, 5000, 1), (40, 151936, 20)])
def test_logprobs_many_rows(qm, typ, T, V, k):
    """A workgroup to a row, and rows in parts."""
    r = rng_of(T, V)
    check(qm, logits(r, T, V, TYPES[typ]), TYPES[typ], r.randint(0, V, T), k)


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("how", ["up", "down", "equal", "two", "zeros", "steps"])
@pytest.mark.parametrize("T,V", [(2, 5000), (1030, 600)])
def test_logprobs_order(qm, typ, how, T, V):
    """Values in an order that keeps the best moving, and equal ones, of which the lowest place is first."""
    r, t, i = rng_of(V), TYPES[typ], np.arange(V)
    x = {"up": i / V * 8, "down": -i / V * 8, "equal": 0 * i + 1.5, "two": i % 2 - 1.0, "zeros": np.where(i % 3, -0.0, 0.0),
         "steps": np.round(3 * r.randn(V))}[how]
    check(qm, np.tile(to_type(x, t), (T, 1)), t, r.randint(0, V, T), 40)


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("T,V", [(3, 5000), (1030, 700)])
def test_logprobs_masked(qm, typ, T, V):
    """Tokens of -inf have no weight; a row may have one token left, or fewer than are asked for."""
    r, t = rng_of(T, 3), TYPES[typ]
    x = 2.5 * r.randn(T, V)
    x[0, :] = -np.inf
    x[0, V - 1] = 3.0
    x[1, :] = -np.inf
    x[1, [5, 77, V // 2]] = [1.0, 2.0, -30.0]
    x[2] = np.where(r.rand(V) < 0.95, -np.inf, x[2])
    token = r.randint(0, V, T)
    token[:2] = V - 1, 3
    x = to_type(x, t)
    lp, ent, ids, val = run(qm, x, t, token, 20)
    assert lp[0] == 0 and ent[0] == 0 and ids[0, 0] == V - 1 and (ids[0, 1:] == np.arange(19)).all()
    assert val[0, 0] == 0 and (val[0, 1:] == -np.inf).all()
    assert lp[1] == -np.inf and list(ids[1, :4]) == [77, 5, V // 2, 0] and (val[1, 3:] == -np.inf).all()
    check(qm, x[1:], t, np.maximum(token[1:], 0), 20)


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("T,V", [(6, 5000), (1030, 300)])
def test_logprobs_not_numbers(qm, typ, T, V):
    """A NaN or +inf, or nothing above -inf: NaN for the row, ids in order, other rows as they were."""
    r, t = rng_of(T, 4), TYPES[typ]
    x, token = logits(r, T, V, t), r.randint(0, V, T)
    plain = run(qm, x, t, token, 10)
    bad = x.copy()
    bad[0, 17] = to_type(np.float32(np.nan), t)
    bad[2, V - 2] = to_type(np.float32(np.inf), t)
    bad[3] = to_type(np.full(V, -np.inf), t)
    bad[4, :] = to_type(np.full(V, np.nan), t)
    bad[4, V - 3] = to_type(np.float32(1.0), t)
    lp, ent, ids, val = run(qm, bad, t, token, 10)
    for i in (0, 2, 3, 4):
        assert np.isnan(lp[i]) and np.isnan(ent[i]) and np.isnan(val[i]).all()
    assert np.array_equal(ids[0], [j for j in order(values(x[0], t)) if j != 17][:10])
    assert ids[2, 0] == V - 2 and np.array_equal(ids[3], np.arange(10)) and list(ids[4]) == [V - 3] + list(range(9))
    keep = [i for i in range(T) if i not in (0, 2, 3, 4)]
    for a, b in zip(plain, (lp, ent, ids, val)):
        assert np.array_equal(a[keep], b[keep])


@pytest.mark.parametrize("T", [4, 1030])
def test_logprobs_tokens(qm, T):
    """Rows without a token have 0, their entropy and alternatives all the same."""
    r = rng_of(T, 5)
    token = r.choice([-1, 0, 299, 300, 2 ** 31 - 1, -2 ** 31], T)
    token[:4] = -1, 0, 299, 300
    check(qm, logits(r, T, 300, F32), F32, token, 4)


@pytest.mark.parametrize("skip", [("logprob",), ("entropy",), ("id", "val"), ("logprob", "entropy"), ("entropy", "id", "val"),
                                  ("logprob", "id", "val"), ("logprob", "entropy", "id", "val")])
def test_logprobs_not_wanted(qm, skip):
    r = rng_of(6)
    for T, V in ((2, 6000), (1030, 300)):
        x, token, k = logits(r, T, V, F32), r.randint(0, V, T), 0 if "id" in skip else 7
        whole = run(qm, x, F32, token, k)
        some = run(qm, x, F32, token, k, skip=skip)
        for n, a, b in zip(("logprob", "entropy", "id", "val"), whole, some):
            assert n in skip or np.array_equal(a, b)


def test_logprobs_far_apart(qm):
    """Logits up to fp32's largest: differences that leave its range are no weight."""
    x = np.zeros((4, 3000), np.float32)
    x[0, :] = -3e38
    x[0, 9] = 3e38
    x[1, :] = -3.4028235e38
    x[2, :] = 1e30
    x[3, 0], x[3, 1:] = 88.0, -20.0
    lp, ent, ids, val = run(qm, x, F32, np.array([9, 5, 7, 0]), 2)
    assert lp[0] == 0 and ent[0] == 0 and ids[0, 0] == 9 and val[0, 1] == -np.inf
    assert np.allclose(lp[1:3], -np.log(3000), rtol=1e-6) and np.allclose(ent[1:3], np.log(3000), rtol=1e-6)
    assert lp[3] == 0 and abs(ent[3]) < 1e-30 or ent[3] >= 0


def test_logprobs_many_small(qm):
    """A token that stands out beside many that are each less than half a step of the sum."""
    V = 151936
    x = np.full((1, V), 0.0, np.float32)
    x[0, 12345] = 17.0           # e^-17 = 0.7 steps of half of 1
    check(qm, x, F32, np.array([12345]), 1)
    check(qm, np.repeat(x, 1030, 0), F32, np.full(1030, 12345), 1)


def test_logprobs_profile(qm):
    r = rng_of(8)
    qm.prof_enable(True)
    run(qm, logits(r, 1, 9000, F32), F32, np.array([3]), 5)
    assert qm.prof_read("logprobs")[0] == 1
    qm.prof_enable(False)
