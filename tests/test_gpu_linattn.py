"""Linear attention with a decay for each head (qmag_linattn_dev), plain and by the delta
rule, against its recurrence in 64 bits."""
import copy

import numpy as np
import pytest

from attn_fixtures import BF16, F16, F32, TYPES, View, to_type, values
from recurrent_fixtures import Sequences, linattn, near, rng_of

pytestmark = pytest.mark.gpu


class Case:
    """Inputs of one call on the host, q, k and v as stored values."""

    def __init__(self, r, s, t, keys=2, heads=4, dk=128, dv=32, delta=True, norm=True, turns=False, decay=True, beta=True):
        self.s, self.t, self.keys, self.heads, self.dk, self.dv = s, t, keys, heads, dk, dv
        self.delta, self.eps, self.turns = delta, 1e-6 if norm else 0.0, turns
        self.q, self.k = (to_type(r.randn(s.rows, keys, dk), t) for _ in range(2))
        self.v = to_type(r.randn(s.rows, heads, dv), t)
        rate = np.exp(r.uniform(np.log(0.005), np.log(4.0), heads))
        self.g = (-rate * np.abs(r.randn(s.rows, heads))).astype(np.float32) if decay else None
        self.b = r.uniform(0, 1, (s.rows, heads)).astype(np.float32) if beta else None
        self.state = (0.3 * r.randn(s.n_slot, heads, dk, dv)).astype(np.float32)
        for i in range(s.n):
            if s.begins(i) and s.keeps(i):
                self.state[s.slots[i]] = np.nan          # what a new sequence's slot holds is not read
        self.scale = dk ** -0.5

    def run(self, qm, layouts=("packed",) * 4, state=None):
        """(out stored, state) of the device; what lies around out is as it was."""
        s, t = self.s, self.t
        q, k, v = (View(qm, x, t, y) for x, y in zip((self.q, self.k, self.v), layouts))
        o = View(qm, np.full((s.rows, self.heads, self.dv), 7, self.v.dtype), t, layouts[3], fill=7)
        state = self.state if state is None else state
        g, b, st = (None if x is None else qm.DBuf.from_array(x) for x in (self.g, self.b, state))
        a = qm.Linattn(self.heads, self.dk, self.dv, int(self.delta), int(self.turns), self.eps, s.n_slot, st.ptr)
        slot, had, cu, n, T = s.args()
        qm.linattn_dev(a, t, q.heads, k.heads, v.heads, o.heads, g and g.ptr, b and b.ptr, slot, had, cu, n, T, self.scale)
        out, same = o.read()
        assert same
        return out, st.download(np.float32).reshape(state.shape)

    def one(self, i, h, S):
        """Sequence i, head h from state S in 64 bits: (out, bound, state, bound)."""
        a, n = self.s.cu[i], self.s.lens[i]
        kh = h % self.keys if self.turns else h // (self.heads // self.keys)
        q, k, v = (values(x[a:a + n, j], self.t) for x, j in ((self.q, kh), (self.k, kh), (self.v, h)))
        g = np.zeros(n) if self.g is None else self.g[a:a + n, h].astype(np.float64)
        b = np.ones(n) if self.b is None else self.b[a:a + n, h].astype(np.float64)
        return linattn(q, k, v, g, b, self.delta, self.eps, S, self.scale, self.dk + 64)

    def check(self, got, after):
        s = self.s
        want = self.state.astype(np.float64)
        seen = np.zeros(s.rows, bool)
        for i in range(s.n):
            a, n = s.cu[i], s.lens[i]
            seen[a:a + n] = True
            if n == 0:
                continue
            for h in range(self.heads):
                S = np.zeros((self.dk, self.dv)) if s.begins(i) else self.state[s.slots[i], h].astype(np.float64)
                out, off, S, e = self.one(i, h, S)
                near(values(got[a:a + n, h], self.t), out, off, self.t, "sequence %d head %d" % (i, h))
                if s.keeps(i):
                    near(after[s.slots[i], h].astype(np.float64), S, e[None] + 1e-30, 0, "state of sequence %d head %d" % (i, h))
                    want[s.slots[i], h] = np.nan
        assert (got[~seen] == 7).all()
        other = ~np.isnan(want) | np.isnan(self.state)
        named = [s.slots[i] for i in range(s.n) if s.keeps(i)]
        left = [j for j in range(s.n_slot) if j not in named]
        assert np.array_equal(after[left], self.state[left], equal_nan=True) and other[left].all()


LENS = {"step": [1] * 7, "some": [3, 1, 0, 9, 16, 2], "edges": [15, 17, 63, 64, 65, 0, 1, 130], "brief": [31, 32, 33, 34, 1, 0], "one": [300], "two": [129, 127]}


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("delta", [True, False])
def test_linattn_lengths(qm, typ, lens, delta):
    r = rng_of(len(lens), delta, 1)
    s = Sequences(qm, r, LENS[lens], pad=3)
    c = Case(r, s, TYPES[typ], delta=delta, norm=delta, beta=delta)
    c.check(*c.run(qm))


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("delta", [True, False])
def test_linattn_many_sequences(qm, typ, delta):
    """More waves than the chip holds at once: 40 rows of 16-bit types go token by token, 96 of fp32."""
    r = rng_of(13, delta)
    s = Sequences(qm, r, [1, 64, 65, 2, 0, 40, 41, 1, 128, 63, 96, 97] + [1] * 30, pad=1)
    c = Case(r, s, TYPES[typ], 4, 8, 64, 64, delta=delta, norm=delta, beta=delta)
    c.check(*c.run(qm))


@pytest.mark.parametrize("typ,least", [("f32", 97), ("bf16", 41)])
def test_linattn_more_walks_than_workgroups(qm, typ, least):
    """4096 walks of 16 columns: a workgroup takes one after another, of sequences with and without values that end one."""
    r = rng_of(14, least)
    s = Sequences(qm, r, [least + 3 * (i % 5) for i in range(16)], pad=1, had="all")
    c = Case(r, s, TYPES[typ], 4, 16, 64, 256)
    c.check(*c.run(qm))
    d = copy.copy(c)
    d.v = c.v.copy()
    d.v[s.cu[3] + 5, 2, 7] = to_type(np.float32(np.inf), TYPES[typ])
    (got, after), (clean, clean_after) = d.run(qm), c.run(qm)
    same = np.ones(got.shape, bool)
    same[s.cu[3] + 5:s.cu[4], 2] = False
    assert np.array_equal(got[same], clean[same])
    others = [j for j in range(s.n_slot) if j != s.slots[3]]
    assert np.array_equal(after[others], clean_after[others], equal_nan=True)


SHAPES = [(1, 1, 64, 16), (2, 6, 64, 48), (3, 3, 128, 128), (1, 4, 128, 144), (2, 2, 256, 64), (1, 2, 256, 256), (5, 5, 64, 112), (1, 6, 64, 32), (2, 18, 64, 16)]


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("keys,heads,dk,dv", SHAPES)
@pytest.mark.parametrize("delta,norm,turns", [(True, True, False), (False, False, True), (False, True, False)])
def test_linattn_heads(qm, typ, keys, heads, dk, dv, delta, norm, turns):
    r = rng_of(keys, dk, dv, delta)
    for lens in ([1, 1, 1], [70, 3, 1]):
        s = Sequences(qm, r, lens, pad=1)
        c = Case(r, s, TYPES[typ], keys, heads, dk, dv, delta, norm, turns, decay=heads != 2, beta=delta or heads == 6)
        c.check(*c.run(qm))


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("lens", [[1, 1, 2], [90, 5]])
@pytest.mark.parametrize("layouts", [("gap", "heads", "odd", "gap"), ("heads", "odd", "gap", "odd"), ("odd", "gap", "heads", "heads")])
def test_linattn_strides(qm, typ, lens, layouts):
    r = rng_of(len(lens), len(layouts[0]), 2)
    s = Sequences(qm, r, lens, pad=2)
    c = Case(r, s, TYPES[typ], 2, 4, 64, 48)
    got, after = c.run(qm, layouts)
    c.check(got, after)
    plain, state = c.run(qm)
    assert np.array_equal(got, plain) and np.array_equal(after, state, equal_nan=True)      # the same sums


@pytest.mark.parametrize("lens", [[1, 1, 1, 1], [80, 2, 64, 1]])
@pytest.mark.parametrize("slots,had", [([-1, 2, 99, 0], "all"), ([5, -1, 1, 3], "all"), ([4, 5, 0, -7], [0, 3, -2, 0])])
def test_linattn_without_state(qm, lens, slots, had):
    r = rng_of(slots[0] + 2, len(lens))
    s = Sequences(qm, r, lens, slots=slots, had=had)
    c = Case(r, s, F32)
    c.check(*c.run(qm))


def test_linattn_no_slots(qm):
    """A call without any state."""
    r = rng_of(3)
    s = Sequences(qm, r, [5, 100], had="all", slots=[-1, -1])
    c = Case(r, s, F32)
    q, k, v = (View(qm, x, F32) for x in (c.q, c.k, c.v))
    o = View(qm, np.full((105, 4, 32), 7, np.float32), F32)
    g, b = qm.DBuf.from_array(c.g), qm.DBuf.from_array(c.b)
    a = qm.Linattn(4, 128, 32, 1, 0, 1e-6, 0, None)
    qm.linattn_dev(a, F32, q.heads, k.heads, v.heads, o.heads, g.ptr, b.ptr, None, None, s.cu_d.ptr, 2, 105, c.scale)
    c.check(o.read()[0], c.state)


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("delta", [True, False])
def test_linattn_in_calls(qm, typ, delta):
    """A prompt cut into calls, down to single tokens, gives what one call gives."""
    t, r = TYPES[typ], rng_of(4, delta)
    s = Sequences(qm, r, [200], slots=[1], had=[0])
    c = Case(r, s, t, delta=delta, norm=delta, beta=delta)
    state, at = c.state, 0
    for n in (1, 130, 2, 1, 1, 20, 45):
        part = Sequences(qm, r, [n], slots=[1], had=[at], spare=2)
        p = Case(r, part, t, delta=delta, norm=delta, beta=delta)
        p.q, p.k, p.v = c.q[at:at + n], c.k[at:at + n], c.v[at:at + n]
        p.g, p.b = c.g[at:at + n], c.b[at:at + n] if delta else None
        out, state = p.run(qm, state=state)
        for h in range(4):
            want, off, S, e = c.one(0, h, np.zeros((128, 32)))
            near(values(out[:, h], t), want[at:at + n], off[at:at + n], t, "tokens from %d" % at)
        at += n
    for h in range(4):
        near(state[1, h].astype(np.float64), c.one(0, h, np.zeros((128, 32)))[2], c.one(0, h, np.zeros((128, 32)))[3][None], 0)


@pytest.mark.parametrize("lens", [[1, 1], [9, 2], [150, 70]])
@pytest.mark.parametrize("delta", [True, False])
def test_linattn_decays(qm, lens, delta):
    """Decays that keep all, forget all, leave fp32's range together, or are above 0 (none)."""
    r = rng_of(len(lens), lens[0], delta)
    s = Sequences(qm, r, lens, had="all")
    c = Case(r, s, F32, 4, 4, 64, 32, delta=delta, norm=delta)
    pick = np.array([0.0, -np.inf, -150.0, 3.0, -1e-6, -40.0, -1e30], np.float32)
    c.g = np.where(r.rand(s.rows, 4) < 0.5, c.g, pick[r.randint(0, 7, (s.rows, 4))]).astype(np.float32)
    c.g[:, 3] = np.where(r.rand(s.rows) < 0.1, np.float32(-np.inf), np.float32(-1e-4))
    c.check(*c.run(qm))


@pytest.mark.parametrize("lens", [[1, 1], [90, 70]])
def test_linattn_keys_alike(qm, lens):
    """The delta rule with keys that repeat, point the other way or are zero, and beta of 0, 1 and 2."""
    r = rng_of(5, lens[0])
    s = Sequences(qm, r, lens)
    c = Case(r, s, F32, 2, 2, 64, 32)
    some = r.randn(3, 64).astype(np.float32)
    c.k = (some[r.randint(0, 3, (s.rows, 2))] * r.choice([-1.0, 1.0, 1.0, 1e-3], (s.rows, 2, 1))).astype(np.float32)
    c.k[5::11] = 0
    c.b = r.choice([0.0, 1.0, 1.0, 2.0], (s.rows, 2)).astype(np.float32)
    c.g[:] = np.where(r.rand(s.rows, 2) < 0.5, 0.0, -1e-3)
    c.check(*c.run(qm))


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("lens", [[3, 2, 4], [150, 70, 100]])
@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("which", ["q", "k", "v", "g", "b", "state"])
def test_linattn_unseen_values(qm, typ, lens, delta, which):
    """NaN and infinities at a token: rows ahead of it, other heads and other sequences have the bits they have
    without; the rest is NaN or infinite where the recurrence has it so."""
    t, r = TYPES[typ], rng_of(lens[0], delta, len(which))
    s = Sequences(qm, r, lens, pad=2, had="all")
    c = Case(r, s, t, 4, 4, 64, 32, delta=delta, norm=delta)
    clean, clean_state = c.run(qm)
    at, h = s.cu[1] + s.lens[1] // 2, 2                # a token of the second sequence
    for bad in (np.nan, np.inf, -np.inf):
        d = Case(rng_of(lens[0], delta, len(which)), s, t, 4, 4, 64, 32, delta=delta, norm=delta)
        d.q, d.k, d.v, d.g, d.b, d.state = (x.copy() for x in (c.q, c.k, c.v, c.g, c.b, c.state))
        if which in "qkv":
            getattr(d, which)[at, h, 5] = to_type(np.float32(bad), t)
        elif which in "gb":
            if which == "g" and bad == -np.inf or which == "b" and not np.isnan(bad) and not delta:
                continue
            getattr(d, which)[at, h] = bad
        else:
            d.state[s.slots[1], h, 3, 4] = bad
        got, state = d.run(qm)
        a0, a1 = s.cu[1], s.cu[2]
        first = a0 if which == "state" else at
        same = np.ones(got.shape, bool)
        same[first:a1, h] = False
        assert np.array_equal(got[same], clean[same])
        held = np.ones(state.shape, bool)
        held[s.slots[1], h] = False
        assert np.array_equal(state[held], clean_state[held])
        want, off, S, _ = d.one(1, h, d.state[s.slots[1], h].astype(np.float64))
        out = values(got[a0:a1, h], t)
        fine = np.isfinite(want) & np.isfinite(off)
        assert np.array_equal(np.isfinite(out), np.isfinite(want)), (which, bad)
        near(np.where(fine, out, 0), np.where(fine, want, 0), np.where(fine, off, 0), t, which)
        assert np.array_equal(np.isfinite(state[s.slots[1], h]), np.isfinite(S))


@pytest.mark.parametrize("lens", [[2, 1], [100, 66]])
@pytest.mark.parametrize("big", [1e4, 1e19, 1e30])
def test_linattn_large_values(qm, lens, big):
    """Values far from 1: v and the state near fp32's range, keys that the norm takes back."""
    r = rng_of(6, lens[0])
    s = Sequences(qm, r, lens, had="all")
    c = Case(r, s, F32, 2, 4, 64, 32)
    c.v = (c.v * np.float32(big)).astype(np.float32)
    c.state = (c.state * np.float32(big)).astype(np.float32)
    c.k = (c.k * np.float32(min(big, 1e16))).astype(np.float32)
    c.check(*c.run(qm))


@pytest.mark.parametrize("lens", [[2, 1], [100, 66]])
def test_linattn_keys_past_norm_one(qm, lens):
    """The delta rule with keys whose b |k|^2 is past 2 grows from token to token; heads within it beside heads that
    are not keep their results."""
    r = rng_of(7, lens[0])
    s = Sequences(qm, r, lens)
    c = Case(r, s, F32, 4, 4, 64, 32, norm=False)
    c.k /= 8
    c.k[:, 2] *= 3
    got, after = c.run(qm)
    calm = Case(rng_of(7, lens[0]), s, F32, 4, 4, 64, 32, norm=False)
    calm.q, calm.k, calm.v, calm.g, calm.b, calm.state = (x.copy() for x in (c.q, c.k, c.v, c.g, c.b, c.state))
    calm.k[:, 2] /= 100
    other, other_after = calm.run(qm)
    keep = [0, 1, 3]
    assert np.array_equal(got[:, keep], other[:, keep])
    assert np.array_equal(after[:, keep], other_after[:, keep], equal_nan=True)
    for i in range(2):
        a = s.cu[i]
        S = np.zeros((64, 32)) if s.begins(i) else c.state[s.slots[i], 2].astype(np.float64)
        want = c.one(i, 2, S)[0]
        n = min(s.lens[i], 4)                     # before the errors grow as the state does
        assert np.allclose(got[a:a + n, 2], want[:n], rtol=1e-3, atol=1e-3 * np.abs(want[:n]).max())


def test_linattn_equal_calls(qm):
    r = rng_of(8)
    for lens in ([1] * 5, [300, 64, 1, 2]):
        s = Sequences(qm, r, lens)
        c = Case(r, s, BF16)
        a, b = c.run(qm), c.run(qm)
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1], equal_nan=True)


def test_linattn_other_sequences(qm):
    """Among calls of the same lengths a sequence's results do not depend on the others' values."""
    r = rng_of(9)
    s = Sequences(qm, r, [70, 130, 5], had="all")
    c = Case(r, s, F32)
    a = c.run(qm)
    c.v[70:200] *= 50
    c.state[s.slots[1]] *= 7
    b = c.run(qm)
    keep = list(range(70)) + list(range(200, 205))
    assert np.array_equal(a[0][keep], b[0][keep]) and np.array_equal(a[1][s.slots[2]], b[1][s.slots[2]])


@pytest.mark.parametrize("delta", [True, False])
def test_linattn_sums_of_any_kind(qm, delta):
    """cu up and down: nothing but rows of out and named states is written."""
    r = rng_of(10)
    s = Sequences(qm, r, [60] * 6, pad=5)
    c = Case(r, s, F32, delta=delta)
    for cu in ([0, 500, -3, 90, 20, 365, 60], [0, 365, 0, 365, 0, 365, 0], [300, 200, 100, 364, -2 ** 31, 2 ** 31 - 1, 5]):
        s.cu_d.upload(np.array(cu, np.int32))
        _, after = c.run(qm, ("packed", "packed", "packed", "gap"))
        other = [i for i in range(s.n_slot) if i not in s.slots]
        assert np.array_equal(after[other], c.state[other])


def test_linattn_profile(qm):
    r = rng_of(11)
    s = Sequences(qm, r, [5])
    c = Case(r, s, F32)
    qm.prof_enable(True)
    c.run(qm)
    assert qm.prof_read("linattn")[0] == 1
    qm.prof_enable(False)


@pytest.mark.parametrize("typ", ["f32", "bf16"])
def test_linattn_windows(qm, typ):
    """A call whose chunks are more than a workspace holds is taken in windows; a sequence that goes on behind one
    hands its state on, with a slot or without."""
    t, r = TYPES[typ], rng_of(12)
    rows = 20000 if typ == "f32" else 30000
    s = Sequences(qm, r, [40, rows - 5000, 1, 300, 4500, 0, 130], pad=1, slots=[3, -1, 1, 0, 2, 5, 4], had="all")
    c = Case(r, s, t, 32, 32, 64, 16)
    got, after = c.run(qm)
    for h in (0, 17):
        for i in range(s.n):
            a, n = s.cu[i], s.lens[i]
            S = c.state[s.slots[i], h].astype(np.float64) if s.slots[i] >= 0 else np.zeros((64, 16))
            out, off, S, e = c.one(i, h, S)
            near(values(got[a:a + n, h], t), out, off, t, "sequence %d head %d" % (i, h))
            if s.keeps(i):
                near(after[s.slots[i], h].astype(np.float64), S, e[None], 0, "state of sequence %d head %d" % (i, h))
    assert (got[-1] == 7).all()
