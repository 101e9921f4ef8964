"""How many bits linear attention (qmag_linattn_dev) holds, token by token and in chunks:
beside the definition in 64 bits and plain fp32 on the same inputs."""
import numpy as np
import pytest

from attn_fixtures import F32, TYPES, values
from linattn_model import near_plain, plain, rounded_as_plain
from recurrent_fixtures import Sequences, linattn, rng_of
from test_gpu_linattn import Case

pytestmark = pytest.mark.gpu


def head(c, h, n):
    """One sequence's head as the forms in numpy take it, and its plain fp32 and 64-bit results."""
    kh = h // (c.heads // c.keys)
    q, k, v = (values(x[:n, j], c.t) for x, j in ((c.q, kh), (c.k, kh), (c.v, h)))
    g = c.g[:n, h].astype(np.float64)
    b = np.ones(n) if c.b is None else c.b[:n, h].astype(np.float64)
    a = (q, k, v, g, b, c.delta, c.eps, c.state[c.s.slots[0], h].astype(np.float64), c.scale)
    want, _, S, _ = linattn(*a, 64)
    return want, S, plain(*a)


@pytest.mark.parametrize("dk", [64, 128, 256])
@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("n", [20, 300])
def test_linattn_fp32_bits(qm, dk, delta, n):
    r = rng_of(dk, delta, n, 21)
    s = Sequences(qm, r, [n], slots=[1], had="all")
    c = Case(r, s, F32, 2, 4, dk, 64, delta=delta, norm=True, beta=delta)
    got, after = c.run(qm)
    for h in range(4):
        want, S, (p, pS) = head(c, h, n)
        near_plain(got[:n, h].astype(np.float64), p, want)
        near_plain(after[1, h].astype(np.float64), pS, S)


@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("dk,dv", [(64, 256), (128, 128), (256, 64)])
@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("n", [20, 600])
def test_linattn_16_bit_results(qm, typ, dk, dv, delta, n):
    """A 16-bit result is rounded once, from fp32: as many results beside the nearest as plain fp32 has."""
    t, r = TYPES[typ], rng_of(dk, delta, n, 22)
    s = Sequences(qm, r, [n], slots=[1], had="all")
    c = Case(r, s, t, 2, 4, dk, dv, delta=delta, norm=True, beta=delta)
    got, after = c.run(qm)
    heads = [head(c, h, n) for h in range(4)]
    rounded_as_plain(got[:n], np.stack([p for _, _, (p, _) in heads], 1), np.stack([w for w, _, _ in heads], 1), t)
    for h, (_, S, (_, pS)) in enumerate(heads):
        near_plain(after[1, h].astype(np.float64), pS, S)
