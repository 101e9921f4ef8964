"""y / (1 + e^-y) of the short convolution (qmag_conv_dev) over all of fp32's range."""
import numpy as np
import pytest

from attn_fixtures import F32
from recurrent_fixtures import Sequences, conv, near, rng_of
from test_gpu_conv import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("W", [2, 4])
def test_conv_silu_range(qm, W):
    """Values down to fp32's smallest normal ones, and results down to them where e^-y is past its largest."""
    y = np.concatenate([2.0 ** np.arange(-125, 20, 0.37), -2.0 ** np.arange(-125, 7, 0.37), np.arange(-93, -60, 0.11), [0.0, -0.0]])
    y = y.astype(np.float32)
    s = Sequences(qm, rng_of(11), [y.size], slots=[0], had=[0])
    w = np.zeros((32, W), np.float32)
    w[:, -1] = 1
    x = np.tile(y[:, None], 32)
    out, _, _ = run(qm, s, x, F32, w, None, True, np.zeros((s.n_slot, W - 1, 32), np.float32))
    want, off, _ = conv(x.astype(np.float64), w.astype(np.float64), 0.0, True, np.zeros((W - 1, 32)))
    # a result has its own rounding below fp32's normal numbers: near allows 1e-38
    near(out, want, off, F32)
