"""Rows of logits with a token that stands alone (qmag_logprobs_dev): what is exact is tested to be."""
import numpy as np
import pytest

from attn_fixtures import BF16, F16, F32, TYPES, to_type, values
from test_gpu_logprobs import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("T", [1, 3, 1030])
@pytest.mark.parametrize("low", [-20.0, -np.inf, "lowest"])
def test_logprobs_one_token(qm, typ, T, low):
    """e^-108 is 0 in fp32, and so are the others' weights below it: a log probability and an entropy of exactly 0."""
    t = TYPES[typ]
    low = {F32: -3.4028235e38, F16: -65504.0, BF16: -3.3895314e38}[t] if low == "lowest" else low
    x = np.full((T, 3000), low)
    at = np.arange(T) * 977 % 3000
    x[np.arange(T), at] = 88.0
    x = to_type(x, t)
    lp, ent, ids, val = run(qm, x, t, at, 2)
    assert (lp == 0).all() and (ent == 0).all()
    assert (ids[:, 0] == at).all() and (val[:, 0] == 0).all()
    assert (ids[:, 1] == (at == 0)).all()                      # the lowest id of the others
    other = values(x[0], t).min() - 88.0
    assert (val[:, 1] == np.float32(other)).all()
