"""Convolution, linear attention and log probabilities as a program runs them: prompts, then
tokens one at a time, then drafts, over states that stay on the device.  q, k and v are views of
the convolution's output, the result goes through a head of weights, the logits are scored.

Each operator is held to its definition in 64 bits on what the device gave it: a wrong view, a
state handed on wrongly or a call that does not wait for the one ahead shows in the next."""
import numpy as np
import pytest

from attn_fixtures import TYPES, ints, store_dtype, to_type, values
from recurrent_fixtures import EPS, Sequences, conv, linattn, near, rng_of

pytestmark = pytest.mark.gpu

KEYS, HEADS, DIM, TAPS, VOCAB, TOP, Q6_K = 2, 4, 64, 4, 515, 5, 14
CHANNELS = (2 * KEYS + HEADS) * DIM


def scored(x, token):
    """Of float64 logits: (log probability, entropy, the best ids, their log probabilities) and how far fp32 may be from
    them: e^(x - m) by its argument's and the difference's rounding, 3 |x - m| 2^-24, and the function's own two; groups of
    eight summed without loss but for a step, then some twenty joins of two roundings each; ln Z and a result rounded."""
    d = x - x.max()
    e = np.exp(d)
    Z = e.sum()
    mean, square, lnz = -(e * d).sum() / Z, (e * d * d).sum() / Z, np.log(e.sum())
    off = (64 + 4 * mean) * EPS
    best = np.argsort(-x, kind="stable")[:TOP]
    p, val = d[token] - lnz, d[best] - lnz
    return ((p, off + 2 * EPS * (abs(p) + lnz)), (lnz + mean, off * (1 + mean) + 4 * EPS * (square + lnz + mean)),
            best, (val, off + 2 * EPS * (np.abs(val) + lnz)))


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("delta", [True, False])
def test_layer_in_calls(qm, typ, delta):
    t, r = TYPES[typ], rng_of(21, delta)
    n_slot, slots = 5, [3, 0, 4]
    taps = (r.randn(CHANNELS, TAPS) / 2).astype(np.float32)
    head = qm.DBuf.from_array((r.randn(VOCAB, HEADS * DIM) / 8).astype(np.float32))
    packed = qm.DBuf(VOCAB * HEADS * DIM // 256 * 210)
    qm.quantize_dev(head.ptr, VOCAB * HEADS * DIM, Q6_K, packed.ptr)
    past = r.randn(n_slot, TAPS - 1, CHANNELS).astype(np.float32)          # junk where sequences begin
    state = r.randn(n_slot, HEADS, DIM, DIM).astype(np.float32)
    taps_d, past_d, state_d = (qm.DBuf.from_array(a) for a in (taps, past, state))
    c = qm.Conv(CHANNELS, TAPS, 1, n_slot, taps_d.ptr, None, past_d.ptr)
    a = qm.Linattn(HEADS, DIM, DIM, int(delta), 0, 1e-6, n_slot, state_d.ptr)
    had = [0, 0, 0]
    for lens in ([150, 40, 0], [1, 1, 1], [3, 1, 5], [1, 90, 0], [1, 1, 1]):
        s = Sequences(qm, r, lens, pad=1, slots=slots, had=had, spare=n_slot - 3)
        T = s.rows
        x = to_type(r.randn(T, CHANNELS), t)
        g = (-np.exp(r.uniform(-5, 1, (T, HEADS)))).astype(np.float32)
        b = r.uniform(0, 1, (T, HEADS)).astype(np.float32)
        token = r.randint(0, VOCAB, T)
        size = np.dtype(store_dtype(t)).itemsize
        x_d, g_d, b_d, mixed, out = (qm.DBuf.from_array(v) for v in (x, g, b, np.zeros_like(x), np.zeros((T, HEADS * DIM), x.dtype)))
        q, k, v = (qm.heads((mixed.ptr + at * DIM * size, n, CHANNELS, DIM)) for at, n in
                   ((0, KEYS), (KEYS, KEYS), (2 * KEYS, HEADS)))
        o = qm.heads((out.ptr, HEADS, HEADS * DIM, DIM))
        args = s.args()
        qm.conv_dev(c, t, x_d.ptr, CHANNELS, mixed.ptr, CHANNELS, *args)
        qm.linattn_dev(a, t, q, k, v, o, g_d.ptr, b_d.ptr, *args, DIM ** -0.5)
        if typ == "f32":
            rows = out
        else:                                      # the head takes fp32
            rows = qm.DBuf.from_array(values(out.download(x.dtype), t).astype(np.float32))
        logits, lp, ent, ids, top = qm.DBuf(4 * T * VOCAB), qm.DBuf(4 * T), qm.DBuf(4 * T), qm.DBuf(4 * T * TOP), qm.DBuf(4 * T * TOP)
        qm.matmul_f32_dev(rows, packed, HEADS * DIM, VOCAB, T, Q6_K, logits)
        tok = ints(qm, token)
        qm.logprobs_dev(VOCAB, 0, logits.ptr, VOCAB, tok.ptr, T, TOP, lp.ptr, ent.ptr, ids.ptr, top.ptr)

        mixed_h = values(mixed.download(x.dtype).reshape(T, CHANNELS), t)
        out_h = values(out.download(x.dtype).reshape(T, HEADS, DIM), t)
        now, after = past_d.download(np.float32).reshape(past.shape), state_d.download(np.float32).reshape(state.shape)
        heads = mixed_h.reshape(T, -1, DIM)
        kept = [slots[i] for i in range(3) if lens[i]]
        for i, n in enumerate(lens):
            if not n:
                continue
            at, sl = slice(s.cu[i], s.cu[i] + n), slots[i]
            y, off, last = conv(values(x[at], t), taps.astype(np.float64), 0.0, True,
                                past[sl].astype(np.float64) if had[i] else np.zeros((TAPS - 1, CHANNELS)))
            near(mixed_h[at], y, off, t, "convolution of sequence %d" % i)
            assert np.array_equal(now[sl].astype(np.float64), last)
            for h in range(HEADS):
                S = state[sl, h].astype(np.float64) if had[i] else np.zeros((DIM, DIM))
                kh = h // (HEADS // KEYS)
                y, off, S, e = linattn(heads[at, kh], heads[at, KEYS + kh], heads[at, 2 * KEYS + h], g[at, h].astype(np.float64),
                                       b[at, h].astype(np.float64), delta, 1e-6, S, DIM ** -0.5, DIM + 64)
                near(out_h[at, h], y, off, t, "sequence %d head %d" % (i, h))
                near(after[sl, h].astype(np.float64), S, e[None] + 1e-30, 0, "state of sequence %d head %d" % (i, h))
        idle = [j for j in range(n_slot) if j not in kept]
        assert np.array_equal(now[idle], past[idle]) and np.array_equal(after[idle], state[idle])
        z = logits.download(np.float32).reshape(T, VOCAB).astype(np.float64)
        lp_h, ent_h, top_h = lp.download(np.float32), ent.download(np.float32), top.download(np.float32).reshape(T, TOP)
        ids_h = ids.download(np.int32).reshape(T, TOP)
        for i in range(T):
            p, h, best, val = scored(z[i], token[i])
            assert abs(lp_h[i] - p[0]) <= p[1] and abs(ent_h[i] - h[0]) <= h[1]
            assert np.array_equal(ids_h[i], best) and (np.abs(top_h[i] - val[0]) <= val[1]).all()
        past, state = now, after
        had = [n0 + n for n0, n in zip(had, lens)]
