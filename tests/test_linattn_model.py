"""What the accuracy tests of linear attention can see, on a model of the chunked form in
numpy: three bf16 parts pass, two fail, whether of all operands or of the results' alone."""
import numpy as np
import pytest

from attn_fixtures import BF16, F16, F32, to_type, values
from linattn_model import chunked, near_plain, plain, rounded_as_plain
from recurrent_fixtures import linattn, rng_of


def inputs(t, n, dk, dv, delta):
    r = rng_of(t, n, dk, delta)
    q, k = (values(to_type(r.randn(n, dk), t), t) for _ in range(2))
    v = values(to_type(r.randn(n, dv), t), t)
    g = (-0.05 * np.abs(r.randn(n))).astype(np.float32).astype(np.float64)
    b = r.uniform(0, 1, n).astype(np.float32).astype(np.float64) if delta else np.ones(n)
    S = (0.3 * r.randn(dk, dv)).astype(np.float32).astype(np.float64)
    return q, k, v, g, b, delta, 1e-6, S, dk ** -0.5


def fails(f, *a):
    with pytest.raises(AssertionError):
        f(*a)


@pytest.mark.parametrize("dk", [64, 128, 256])
@pytest.mark.parametrize("delta", [True, False])
def test_three_parts_are_seen(dk, delta):
    a = inputs(F32, 300, dk, 64, delta)
    want, _, S, _ = linattn(*a, 64)
    p, pS = plain(*a)
    three, two, out_two = chunked(*a, 3, 3), chunked(*a, 2, 2), chunked(*a, 3, 2)
    near_plain(three[0], p, want)
    near_plain(three[1], pS, S)
    fails(near_plain, two[0], p, want)
    fails(near_plain, two[1], pS, S)
    fails(near_plain, out_two[0], p, want)


@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("delta", [True, False])
def test_results_of_16_bits(t, delta):
    a = inputs(t, 600, 128, 256, delta)
    want, _, S, _ = linattn(*a, 64)
    p, pS = plain(*a)
    three, two = chunked(*a, 3, 3), chunked(*a, 3, 2)
    rounded_as_plain(to_type(three[0], t), p, want, t)
    fails(rounded_as_plain, to_type(two[0], t), p, want, t)
    near_plain(three[1], pS, S)
