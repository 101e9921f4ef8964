"""Linear attention of one head in numpy: token by token in plain fp32, and in chunks with
the products' operands cut to a number of bf16 parts, as the matrix cores take them.  What
the accuracy tests compare with."""
import numpy as np

from attn_fixtures import BF16, F16, to_type, values


def plain(q, k, v, g, b, delta, eps, S, scale):
    """The recurrence in fp32 throughout, a token after another: (out, state) in float32."""
    f = np.float32
    q, k, v, g, b, S = (x.astype(f) for x in (q, k, v, g, b, S))
    out = np.zeros(v.shape, f)
    for t in range(q.shape[0]):
        kt, qt = k[t], q[t]
        if eps > 0:
            kt, qt = kt * (f(1) / np.sqrt(kt @ kt + f(eps))), qt * (f(1) / np.sqrt(qt @ qt + f(eps)))
        S = S * np.exp(g[t])
        u = b[t] * (v[t] - kt @ S) if delta else b[t] * v[t]
        S = S + kt[:, None] * u
        out[t] = f(scale) * (qt @ S)
    return out, S


def parts(x, n):
    """x as the sum of n bf16 numbers, each the nearest to what those ahead leave."""
    r, got = np.asarray(x, np.float32), np.zeros(np.shape(x), np.float32)
    for _ in range(n):
        p = values(to_type(r, BF16), BF16).astype(np.float32)
        got, r = got + p, r - p
    return got.astype(np.float64)


def chunked(q, k, v, g, b, delta, eps, S, scale, n, n_out, chunk=64):
    """In chunks, all but the operands in 64 bits: the state, X, U and the triangle's inverse
    as n parts each, and n_out of U, P and the state where only a result is made of them."""
    f = np.float64
    q, k = q.astype(f), k.astype(f)
    out = np.zeros(v.shape)
    S = S.astype(np.float32)
    for a in range(0, q.shape[0], chunk):
        s = slice(a, min(a + chunk, q.shape[0]))
        qc, kc, vc, bc, G = q[s], k[s], v[s], b[s], np.cumsum(g[s])
        if eps > 0:
            qc, kc = (x / np.sqrt((x * x).sum(1, keepdims=True) + eps) for x in (qc, kc))
        since = np.exp(np.minimum(G[:, None] - G[None], 0.0))
        x = bc[:, None] * (vc - np.exp(G)[:, None] * (kc @ parts(S, n)) if delta else vc)
        if delta:
            L = bc[:, None] * (kc @ kc.T) * since * np.tri(len(G), k=-1)
            u = (parts(np.linalg.inv(np.eye(len(G)) + L), n) @ parts(x, n)).astype(np.float32)
        else:
            u = x.astype(np.float32)
        P = scale * (qc @ kc.T) * since * np.tri(len(G))
        out[s] = scale * np.exp(G)[:, None] * (qc @ parts(S, n_out)) + parts(P, n_out) @ parts(u, n_out)
        S = (np.exp(G[-1]) * S + kc.T @ parts(np.exp(G[-1] - G)[:, None] * u, n)).astype(np.float32)
    return out, S


def rms(got, want):
    """The root of the mean squared difference, relative to that of the values."""
    return np.sqrt(((got - want) ** 2).sum() / (want ** 2).sum())


# How far the device may be from the definition in 64 bits, measured by how far plain fp32 on
# the same inputs is.  Three bf16 parts hold 2^-25 of an operand and the products left out
# 2^-24, as many roundings as plain fp32's own sums have, or fewer: three times its error
# leaves room for sums in another order.  Two parts hold 2^-17, and are ten times and more off.
TIMES = 3.0


def near_plain(got, plain_got, want):
    """fp32 values: within TIMES the plain fp32 form's error."""
    assert rms(got, want) <= TIMES * rms(plain_got.astype(np.float64), want) + 2.0 ** -24, (rms(got, want), rms(plain_got, want))


def misrounded(got, want, t):
    """How many stored values of a 16-bit type are not what rounding `want` gives."""
    return int((values(got, t) != values(to_type(want, t), t)).sum())


def rounded_as_plain(got, plain_got, want, t):
    """16-bit values: a result whose error is e ahead of its rounding falls to the other side of a border
    in a share of cases that grows with e, so that counting them shows e below the rounding.  TIMES the
    plain form's count, three standard deviations of a count and three more."""
    mine, n = misrounded(got, want, t), misrounded(to_type(plain_got, t), want, t)
    assert mine <= TIMES * (n + 3.0 * np.sqrt(n) + 3.0), (mine, n, want.size)
