"""What the tests of the recurrent layers' entries share: packed sequences on the device,
the operators' definitions in 64 bits, and how far fp32 may be from them."""
import numpy as np

from attn_fixtures import HALF, View, ints, to_type, values

EPS = 2.0 ** -24


def rng_of(*seed):
    return np.random.RandomState([int(s) % (1 << 31) for s in seed])


class Sequences:
    """Packed sequences of the given lengths, each with a slot and a count of tokens before."""

    def __init__(self, qm, r, lens, pad=0, slots=None, had=None, spare=2):
        self.lens = list(lens)
        self.n = len(lens)
        self.cu = np.concatenate([[0], np.cumsum(lens)]).astype(int)
        self.rows = int(self.cu[-1]) + pad
        self.n_slot = self.n + spare
        self.slots = list(r.permutation(self.n_slot)[:self.n]) if slots is None else list(slots)
        self.had = [int(x) for x in r.randint(0, 2, self.n) * 7] if had is None else had
        self.cu_d, self.slot_d = ints(qm, self.cu), ints(qm, self.slots)
        self.len_d = None if self.had == "all" else ints(qm, self.had)

    def begins(self, i):
        """whether sequence i begins from nothing"""
        return not 0 <= self.slots[i] < self.n_slot or (self.had != "all" and self.had[i] <= 0)

    def keeps(self, i):
        return self.lens[i] > 0 and 0 <= self.slots[i] < self.n_slot

    def args(self):
        return self.slot_d.ptr, self.len_d.ptr if self.len_d else None, self.cu_d.ptr, self.n, self.rows


# -------------------------------------------------------------------- conv --

def conv(x, weight, bias, silu, past):
    """x [n][C] float64, past [W - 1][C]: (out, what W products and sums may be off by, the state behind it)."""
    n, W = x.shape[0], weight.shape[1]
    a = np.concatenate([past, x])
    y, mag = np.zeros(x.shape) + bias, np.zeros(x.shape) + np.abs(bias)
    for w in range(W):
        y += a[w:w + n] * weight[:, w]
        mag += np.abs(a[w:w + n] * weight[:, w])
    off = (W + 1) * EPS * mag
    if silu:
        with np.errstate(over="ignore"):
            s = 1.0 / (1.0 + np.exp(-y))
        # a slope of at most 1.1; e^-y, the sum, the quotient: two units in the last place each, e^-y's own
        # rounding of its argument |y| 2^-24
        y, off = y * s, 1.1 * off + np.abs(y * s) * (6 + np.abs(y)) * EPS
    return y, off, a[n:]


# ----------------------------------------------------------------- linattn --

def linattn(q, k, v, g, b, delta, eps, S, scale, terms):
    """One head: q, k [n][dk], v [n][dv], g, b [n], S [dk][dv] float64.  Returns (out, its bound, S, its
    bound).

    The bound: a dot product of fp32 numbers, in any order of at most `terms` additions, is off by terms
    2^-24 |x||y|, and each further rounding by 2^-24 of a value.  A column s of the state has
    e <- a |I - b k k^T| e + (terms + 4) 2^-24 (|s| + |k||u|), where for keys of norm 1 and b of 0 to 2 (and
    without the delta rule) the factor's norm is at most 1, and a result scale |q| e + terms 2^-24 scale |q||s|."""
    n, dv = q.shape[0], v.shape[1]
    out, off = np.zeros((n, dv)), np.zeros((n, dv))
    S, e = S.copy(), np.zeros(dv)
    u_rel = (terms + 8) * EPS
    with np.errstate(all="ignore"):
        for t in range(n):
            kt, qt = k[t], q[t]
            if eps > 0:
                kt, qt = kt / np.sqrt(kt @ kt + eps), qt / np.sqrt(qt @ qt + eps)
            a, nk, nq = np.exp(min(g[t], 0.0) if g[t] == g[t] else g[t]), np.sqrt(kt @ kt), np.sqrt(qt @ qt)
            S = S * a
            was = np.sqrt((S * S).sum(0))
            u = b[t] * (v[t] - kt @ S) if delta else b[t] * v[t]
            S = S + kt[:, None] * u
            now = np.sqrt((S * S).sum(0))
            e = a * e + u_rel * (was + now + nk * (np.abs(u) + abs(b[t]) * (np.abs(v[t]) + nk * was * delta)))
            out[t] = scale * (qt @ S)
            off[t] = abs(scale) * nq * (e + u_rel * (was + now + nk * np.abs(u)))
    return out, off, S, e


def near(got, want, off, t, what=""):
    """got (stored values of type t, as float64) is want rounded once, give or take off."""
    tol = off + (HALF[t] if t else 2.0 ** -24) * (np.abs(want) + off) + (2.0 ** -25 if t == 1 else 1e-38)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), "%s: %d of %d off, first %r: %r for %r, tolerance %r" % (
        what, bad.sum(), bad.size, np.argwhere(bad)[0], got[bad][0], want[bad][0], tol[bad][0])
