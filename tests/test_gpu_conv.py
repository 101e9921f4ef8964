"""Short causal convolution (qmag_conv_dev) against its definition in 64 bits."""
import numpy as np
import pytest

from attn_fixtures import BF16, F16, F32, TYPES, View, to_type, values
from recurrent_fixtures import Sequences, conv, near, rng_of

pytestmark = pytest.mark.gpu


def run(qm, s, x, t, weight, bias, silu, state, xlayout="packed", olayout="packed"):
    """x [rows][C] stored: (out stored, rows behind the last sequence and gaps as they were, state)."""
    C, W = weight.shape
    vx = View(qm, x[:, None], t, xlayout)
    vo = View(qm, np.full(x[:, None].shape, 7, x.dtype), t, olayout, fill=7)
    wb, bb, sb = qm.DBuf.from_array(weight), None if bias is None else qm.DBuf.from_array(bias), qm.DBuf.from_array(state)
    c = qm.Conv(C, W, int(silu), state.shape[0], wb.ptr, bb.ptr if bb else None, sb.ptr)
    slot, had, cu, n, T = s.args()
    hx, ho = vx.heads[0], vo.heads[0]
    qm.conv_dev(c, t, hx.ptr, hx.token_stride, ho.ptr, ho.token_stride, slot, had, cu, n, T)
    out, same = vo.read()
    return out[:, 0], same, sb.download(np.float32).reshape(state.shape)


def check(qm, s, r, t, C, W, silu, bias, xlayout="packed", olayout="packed", x=None):
    x = to_type(r.randn(s.rows, C) if x is None else x, t)
    weight = (r.randn(C, W) / 2).astype(np.float32)
    b = (r.randn(C) / 2).astype(np.float32) if bias else None
    state = r.randn(s.n_slot, W - 1, C).astype(np.float32)
    for i in range(s.n):
        if s.begins(i) and s.keeps(i):
            state[s.slots[i]] = np.nan                  # what a new sequence's slot holds is not read
    out, same, after = run(qm, s, x, t, weight, b, silu, state, xlayout, olayout)
    assert same
    want_state = state.astype(np.float64)
    seen = np.zeros(s.rows, bool)
    for i in range(s.n):
        a, n = s.cu[i], s.lens[i]
        past = np.zeros((W - 1, C)) if s.begins(i) else state[s.slots[i]].astype(np.float64)
        y, off, last = conv(values(x[a:a + n], t), weight.astype(np.float64), 0.0 if b is None else b.astype(np.float64), silu, past)
        near(values(out[a:a + n], t), y, off, t, "sequence %d" % i)
        seen[a:a + n] = True
        if s.keeps(i):
            want_state[s.slots[i]] = last
    assert (out[~seen] == 7).all()
    assert np.array_equal(after.astype(np.float64), want_state, equal_nan=True)      # inputs, held exactly
    return out


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("C", [1, 7, 64, 260, 1030])
def test_conv_shapes(qm, typ, W, C):
    r = rng_of(W, C, 1)
    s = Sequences(qm, r, [1, 0, 2, 3, 4, 5, 31, 1, 33, 70], pad=3)
    check(qm, s, r, TYPES[typ], C, W, C % 2 == 1, W != 3)


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("lens", [[1], [1] * 9, [4096], [1000, 0, 0, 2], [4] * 40])
def test_conv_lengths(qm, typ, lens):
    r = rng_of(len(lens), lens[0], 2)
    check(qm, Sequences(qm, r, lens, pad=1), r, TYPES[typ], 512, 4, True, False)


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("xl,ol", [("gap", "odd"), ("odd", "gap"), ("odd", "odd")])
def test_conv_strides(qm, typ, xl, ol):
    r = rng_of(3, len(xl))
    check(qm, Sequences(qm, r, [9, 1, 40], pad=2), r, TYPES[typ], 100, 4, True, True, xl, ol)


@pytest.mark.parametrize("slots", [[-1, 2, 99, 0], [5, -1, -1, 3]])
def test_conv_without_state(qm, slots):
    r = rng_of(4, slots[0] + 2)
    check(qm, Sequences(qm, r, [3, 50, 2, 1], slots=slots, had="all"), r, F32, 96, 4, True, True)


def test_conv_no_slots(qm):
    """A call without any state."""
    r = rng_of(5)
    s = Sequences(qm, r, [3, 20], had="all")
    x = r.randn(23, 64).astype(np.float32)
    w = r.randn(64, 4).astype(np.float32)
    xb, wb, ob = qm.DBuf.from_array(x), qm.DBuf.from_array(w), qm.DBuf(4 * x.size)
    c = qm.Conv(64, 4, 0, 0, wb.ptr, None, None)
    qm.conv_dev(c, F32, xb.ptr, 64, ob.ptr, 64, None, None, s.cu_d.ptr, 2, 23)
    got = ob.download(np.float32).reshape(x.shape)
    for a, n in ((0, 3), (3, 20)):
        y, off, _ = conv(x[a:a + n].astype(np.float64), w.astype(np.float64), 0.0, False, np.zeros((3, 64)))
        near(got[a:a + n], y, off, F32)


@pytest.mark.parametrize("typ", TYPES)
def test_conv_in_calls(qm, typ):
    """A prompt cut into calls, down to single tokens, gives the bits of one call."""
    t, r = TYPES[typ], rng_of(6)
    C, W = 200, 4
    w, x = r.randn(C, W).astype(np.float32), to_type(r.randn(90, C), t)
    one = Sequences(qm, r, [90], slots=[1], had=[0])
    state = np.zeros((3, W - 1, C), np.float32)
    whole, _, end = run(qm, one, x, t, w, None, True, state)
    at, parts = 0, []
    for n in (1, 1, 2, 3, 40, 5, 38):
        s = Sequences(qm, r, [n], slots=[1], had=[at])
        s.n_slot = 3
        out, _, state = run(qm, s, x[at:at + n], t, w, None, True, state)
        parts.append(out)
        at += n
    assert np.array_equal(np.concatenate(parts), whole) and np.array_equal(state[1], end[1])


def test_conv_unseen_values(qm):
    """NaN and infinities reach the W - 1 tokens behind them in their channel, no others, no other sequence."""
    r = rng_of(7)
    s = Sequences(qm, r, [40, 6, 30], pad=2, had=[0, 0, 0])
    C, W = 64, 4
    w = r.randn(C, W).astype(np.float32)
    x = r.randn(s.rows, C).astype(np.float32)
    state = np.zeros((s.n_slot, W - 1, C), np.float32)
    clean, _, _ = run(qm, s, x, F32, w, None, True, state)
    bad = x.copy()
    bad[10, 5], bad[39, 6], bad[76:, :] = np.nan, np.inf, np.nan
    got, _, after = run(qm, s, bad, F32, w, None, True, state)
    reach = np.zeros(x.shape, bool)
    reach[10:14, 5] = reach[39, 6] = True
    reach[76:] = True
    assert np.array_equal(got[~reach], clean[~reach])
    assert np.isnan(got[10:14, 5]).all() and not np.isfinite(got[39, 6])
    assert np.isinf(after[s.slots[0], 2, 6]) and np.isfinite(after[s.slots[1:]]).all()


def test_conv_large_values(qm):
    """e^-y past fp32's range: 0 or y, never NaN."""
    r = rng_of(8)
    x = np.array([-1e38, -3e4, -200.0, -100.0, -88.0, 0.0, 88.0, 1e38])
    s = Sequences(qm, r, [8], had=[0])
    w = np.tile(np.float32([0, 0, 0, 1]), (16, 1))
    out, _, _ = run(qm, s, to_type(np.tile(x[:, None], 16), F32), F32, w, None, True, np.zeros((s.n_slot, 3, 16), np.float32))
    with np.errstate(over="ignore"):
        want = x / (1 + np.exp(-x.astype(np.float64)))
    assert np.isfinite(out).all() and np.allclose(out[:, 0], want, rtol=1e-5, atol=1e-37)


def test_conv_sums_of_any_kind(qm):
    """cu up and down: nothing but rows of out and named states is written."""
    r = rng_of(9)
    s = Sequences(qm, r, [30] * 6, pad=5)
    s.cu_d.upload(np.array([0, 500, -3, 90, 20, 185, 60], np.int32))
    w = r.randn(48, 4).astype(np.float32)
    state = r.randn(s.n_slot, 3, 48).astype(np.float32)
    out, same, after = run(qm, s, r.randn(s.rows, 48).astype(np.float32), F32, w, None, True, state, "gap", "gap")
    assert same and np.isfinite(out).all()
    other = [i for i in range(s.n_slot) if i not in s.slots]
    assert np.array_equal(after[other], state[other])


def test_conv_profile(qm):
    r = rng_of(10)
    s = Sequences(qm, r, [5])
    qm.prof_enable(True)
    run(qm, s, r.randn(5, 16).astype(np.float32), F32, r.randn(16, 4).astype(np.float32), None, True, np.zeros((s.n_slot, 3, 16), np.float32))
    assert qm.prof_read("conv")[0] == 1
    qm.prof_enable(False)
