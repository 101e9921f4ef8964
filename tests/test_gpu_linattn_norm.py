"""Linear attention of keys and queries whose squares leave fp32's range, with the norm that takes them back."""
import numpy as np
import pytest

from attn_fixtures import BF16, F32, to_type
from recurrent_fixtures import Sequences, rng_of
from test_gpu_linattn import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("lens", [[1, 3], [33, 20], [150, 70]])
@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("big", [1e19, 1e25, 7e37])
def test_linattn_keys_past_squares(qm, t, lens, delta, big):
    """One token of each sequence, of q and of k, then every token."""
    for rows in (slice(lens[0] - 1, lens[0] + 1), slice(None)):
        r = rng_of(41, lens[0], delta)
        s = Sequences(qm, r, lens, had="all")
        c = Case(r, s, F32, 2, 4, 64, 32, delta=delta)
        c.k[rows] *= np.float32(big)
        c.q[rows] *= np.float32(big)
        c.t = t
        c.q, c.k, c.v = (to_type(np.clip(x, -3e38, 3e38), t) for x in (c.q, c.k, c.v))
        c.check(*c.run(qm))
