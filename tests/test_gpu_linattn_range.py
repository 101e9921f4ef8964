"""Linear attention of values that a chunk's products would leave fp32's range with: the
results are those of the recurrence, however long the sequence is."""
import numpy as np
import pytest

from attn_fixtures import F32
from recurrent_fixtures import Sequences, rng_of
from test_gpu_linattn import Case

pytestmark = pytest.mark.gpu

LENS = [[3, 1], [33, 20], [64, 100], [200, 70]]


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("key,state", [(1e10, 1e28), (1e11, 1e29), (1e3, 1e30), (1e11, 1e20)])
def test_linattn_keys_and_state(qm, lens, key, state):
    """Keys and queries that the norm takes back, against a state: their products ahead of it reach 2^137."""
    r = rng_of(31, lens[0], int(np.log10(key * state)))
    s = Sequences(qm, r, lens, pad=1, had="all")
    c = Case(r, s, F32, 2, 4, 64, 32)
    c.q, c.k, c.state = (x * np.float32(y) for x, y in ((c.q, key), (c.k, key), (c.state, state)))
    c.check(*c.run(qm))


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("norm", [True, False])
def test_linattn_state_that_grows(qm, lens, norm):
    """A plain sum whose state leaves what a chunk's products hold after the first chunk, or with the last one."""
    r = rng_of(32, lens[0], norm)
    s = Sequences(qm, r, lens, had="all")
    c = Case(r, s, F32, 2, 4, 64, 32, delta=False, norm=norm)
    c.g[:] = -1e-3
    c.v = (np.abs(c.v) * np.float32(2.0 ** 39)).astype(np.float32)
    c.b = np.full(c.b.shape, 2.0 ** 19, np.float32)
    c.k = (np.abs(c.k) * np.float32(2.0 ** (30 if norm else 16))).astype(np.float32)
    c.state = (c.state * np.float32(2.0 ** (92 if norm else 78))).astype(np.float32)
    c.q = (c.q * np.float32(2.0 ** (36 if norm else 16))).astype(np.float32)
    c.check(*c.run(qm))


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("delta", [True, False])
def test_linattn_large_gates_and_values(qm, lens, delta):
    """beta and v that only together leave the range that a chunk's products hold, at one token and at all of them."""
    for rows in (slice(lens[0] // 2, lens[0] // 2 + 1), slice(None)):
        r = rng_of(33, lens[0], delta)
        s = Sequences(qm, r, lens, had="all")
        c = Case(r, s, F32, 2, 4, 64, 32, delta=delta, norm=delta)
        c.v, c.b, c.k = c.v.copy(), c.b.copy(), c.k.copy()
        c.v[rows] *= np.float32(2.0 ** 58)
        if delta:
            c.k[rows] *= np.float32(2.0 ** -38)           # eps is most of such a key's square
            c.b[rows] *= np.float32(2.0 ** 19)
        else:
            c.b[rows] *= np.float32(2.0 ** 38)
        c.check(*c.run(qm))


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("scale", [2.0 ** 60, 2.0 ** -100, 0.0, -3.0])
def test_linattn_scales(qm, lens, scale):
    r = rng_of(34, lens[0])
    s = Sequences(qm, r, lens, had="all")
    c = Case(r, s, F32, 2, 4, 64, 32)
    c.scale = scale
    c.check(*c.run(qm))


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("eps", [2.0 ** -120, 2.0 ** -140])
def test_linattn_no_key(qm, lens, eps):
    """Keys and queries of zeros, whose norm is the smallest eps'."""
    r = rng_of(35, lens[0])
    s = Sequences(qm, r, lens, had="all")
    c = Case(r, s, F32, 2, 4, 64, 32)
    c.eps = eps
    c.k[::3], c.q[1::3] = 0, 0
    c.v = c.v * np.float32(2.0 ** 39)
    c.check(*c.run(qm))


def test_linattn_rows_ahead_of_large_ones(qm):
    """A finite value that ends a chunk's walk leaves the rows ahead of it as accurate as they are without."""
    r = rng_of(36)
    s = Sequences(qm, r, [190], had="all")
    for what, value in (("v", 1e37), ("b", 1e30), ("k", 1e18), ("q", 1e18)):
        c = Case(rng_of(37), s, F32, 2, 4, 64, 32, delta=what != "b", norm=what != "b")
        x = getattr(c, what)
        x[100, 1] = np.float32(value)
        c.check(*c.run(qm))


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("norm", [True, False])
def test_linattn_small_keys(qm, lens, norm):
    """Keys whose squares are below fp32's smallest number, and whose products with a large v are not."""
    r = rng_of(38, lens[0], norm)
    s = Sequences(qm, r, lens, had=[0] * len(lens))
    c = Case(r, s, F32, 2, 4, 64, 32, delta=False, norm=norm, beta=False)
    c.k = (c.k * np.float32(2.0 ** -85)).astype(np.float32)
    c.v = (c.v * np.float32(2.0 ** 38)).astype(np.float32)
    c.check(*c.run(qm))
