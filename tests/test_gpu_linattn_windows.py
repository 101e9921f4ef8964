"""Linear attention (qmag_linattn_dev) of calls that its workspace takes in several windows: a sequence that goes on
behind one hands its state over.  Many heads over broadcast q, k and v make a window of some hundred rows."""
import numpy as np
import pytest

from attn_fixtures import BF16, F16, F32, TYPES, View, to_type, values
from linattn_plan import windows
from recurrent_fixtures import Sequences, linattn, near, rng_of

pytestmark = pytest.mark.gpu

HEADS, DV, ROWS = 256, 16, 3000
PARTS = {F32: 3, F16: 2, BF16: 1}


class Wide:
    """One q, k and v for all heads, gates for each: sequences cut where windows end."""

    def __init__(self, qm, t, delta, dk, n_seq=4, slots=(3, 1, 0, 2)):
        r = rng_of(t, delta, dk, 51)
        (self.window, _, self.brief), = windows([(ROWS, n_seq, HEADS, HEADS, dk, DV, PARTS[t])])
        self.n_windows = -(-ROWS // self.window)
        assert self.n_windows >= 3
        # the second sequence ends in the last window but one, a few rows behind its border; the third begins there
        last = (self.n_windows - 1) * self.window
        end = last + 20 if ROWS - last > 140 else last - self.window + 20
        lens = [100, end - 100, ROWS - 7 - end, 7] if n_seq == 4 else [ROWS]
        self.s = Sequences(qm, r, lens, pad=0, slots=list(slots)[:n_seq], had="all")
        self.t, self.delta, self.dk, self.eps, self.scale = t, delta, dk, 1e-6, dk ** -0.5
        self.q, self.k = (to_type(r.randn(ROWS, dk), t) for _ in range(2))
        self.v = to_type(r.randn(ROWS, DV), t)
        rate = np.exp(r.uniform(np.log(0.005), np.log(0.5), HEADS))
        self.g = (-rate * np.abs(r.randn(ROWS, HEADS))).astype(np.float32)
        self.b = r.uniform(0, 1, (ROWS, HEADS)).astype(np.float32)
        self.state = (0.3 * r.randn(self.s.n_slot, HEADS, dk, DV)).astype(np.float32)

    def run(self, qm):
        q, k, v, g, b, st = (qm.DBuf.from_array(x) for x in (self.q, self.k, self.v, self.g, self.b, self.state))
        o = View(qm, np.full((ROWS, HEADS, DV), 7, self.v.dtype), self.t, fill=7)
        hq, hk, hv = (qm.heads((x.ptr, HEADS, n, 0)) for x, n in ((q, self.dk), (k, self.dk), (v, DV)))
        a = qm.Linattn(HEADS, self.dk, DV, int(self.delta), 0, self.eps, self.s.n_slot, st.ptr)
        slot, had, cu, n, T = self.s.args()
        qm.linattn_dev(a, self.t, hq, hk, hv, o.heads, g.ptr, b.ptr, slot, had, cu, n, T, self.scale)
        return o.read()[0], st.download(np.float32).reshape(self.state.shape)

    def one(self, i, h):
        a, n = self.s.cu[i], self.s.lens[i]
        x = [values(y[a:a + n], self.t) for y in (self.q, self.k, self.v)]
        S = self.state[self.s.slots[i], h].astype(np.float64) if self.s.keeps(i) else np.zeros((self.dk, DV))
        return linattn(*x, self.g[a:a + n, h].astype(np.float64), self.b[a:a + n, h].astype(np.float64), self.delta, self.eps, S,
                       self.scale, self.dk + 64)

    def check(self, got, after, heads=(0, 255), finite=True):
        for i in range(self.s.n):
            a, n = self.s.cu[i], self.s.lens[i]
            for h in heads:
                out, off, S, e = self.one(i, h)
                x, y = values(got[a:a + n, h], self.t), after[self.s.slots[i], h].astype(np.float64) if self.s.keeps(i) else None
                if not finite:
                    assert np.array_equal(np.isfinite(x), np.isfinite(out))
                    fine = np.isfinite(out) & np.isfinite(off)
                    x, out, off = (np.where(fine, z, 0) for z in (x, out, off))
                near(x, out, off, self.t, "sequence %d head %d" % (i, h))
                if y is not None:
                    if not finite:
                        assert np.array_equal(np.isfinite(y), np.isfinite(S))
                        fine = np.isfinite(S) & np.isfinite(e)[None]
                        y, S, e = np.where(fine, y, 0), np.where(fine, S, 0), np.where(np.isfinite(e), e, 0)
                    near(y, S, e[None] + 1e-30, 0, "state of sequence %d head %d" % (i, h))


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("delta", [True, False])
def test_linattn_three_windows(qm, typ, delta):
    """Two sequences over borders, one of them ending a few rows behind its last, with a slot each."""
    c = Wide(qm, TYPES[typ], delta, 256)
    got, after = c.run(qm)
    c.check(got, after)
    others = [j for j in range(c.s.n_slot) if j not in c.s.slots]
    assert np.array_equal(after[others], c.state[others])


@pytest.mark.parametrize("delta", [True, False])
def test_linattn_windows_without_slots(qm, delta):
    """A state that no slot has is handed over all the same."""
    c = Wide(qm, F32, delta, 256, slots=(3, -1, 99, 2))
    got, after = c.run(qm)
    c.check(got, after)


@pytest.mark.parametrize("typ", ["f32", "bf16"])
@pytest.mark.parametrize("delta", [True, False])
def test_linattn_windows_of_one_sequence(qm, typ, delta):
    """A walk over all windows, each state from the one before."""
    c = Wide(qm, TYPES[typ], delta, 256, n_seq=1, slots=(1,))
    got, after = c.run(qm)
    c.check(got, after, heads=(3,))


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("value", [np.nan, np.inf, 1e30])
def test_linattn_values_in_a_later_window(qm, delta, value):
    """A value that ends the walk of the second window: that window goes token by token from the state handed over, rows
    ahead of it and other sequences keep their bits."""
    c = Wide(qm, F32, delta, 256)
    clean, clean_after = c.run(qm)
    at = c.window + 70
    c.v[at, 5] = np.float32(value)
    got, after = c.run(qm)
    same = np.ones(ROWS, bool)
    same[at:c.s.cu[2]] = False
    assert c.s.cu[1] < at < c.s.cu[2] and np.array_equal(got[same], clean[same])
    other = [c.s.slots[i] for i in (0, 2, 3)]
    assert np.array_equal(after[other], clean_after[other])
    c.check(got, after, heads=(17,), finite=False)
