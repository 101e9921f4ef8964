"""The attention entries against plain 64-bit forms: rotary positions, the paged
4-bit cache and its bookkeeping, attention over the cache and over prompts."""
import numpy as np
import pytest

from attn_fixtures import (BF16, F16, F32, HALF, TYPES, View, attention, block_bytes, held, ints, quantise, rope, to_type,
                           values)

pytestmark = pytest.mark.gpu


def rng_of(*a):
    return np.random.RandomState(sum((i + 1) * 7919 * int(x) for i, x in enumerate(a)) % (1 << 31))


def close(got, want, tol, what=""):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:3].tolist(),
                           float(np.max(np.where(bad, np.abs(got - want) / tol, 0))))


# -------------------------------------------------------------------- rope --

@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("T,H,KV,D,rot,sections,turns,adjacent,layout", [
    (1, 16, 2, 256, 64, (11, 11, 10), True, False, "packed"),
    (7, 4, 1, 128, 128, (16, 24, 24), False, False, "gap"),
    (33, 3, 3, 64, 32, (16,), False, True, "heads"),
    (5, 2, 1, 80, 20, (4, 1, 2, 3), True, True, "odd"),
    (9, 5, 1, 96, 96, (0, 40, 8), True, False, "odd"),
    (3, 1, 1, 6, 2, (1,), False, False, "packed"),
    (300, 8, 8, 64, 64, (8, 0, 24), True, True, "packed"),
    (2, 70, 2, 1024, 256, (128,), False, False, "packed"),
])
def test_rope(qm, typ, T, H, KV, D, rot, sections, turns, adjacent, layout):
    t = TYPES[typ]
    r = rng_of(T, H, D)
    theta = 1e4
    pos = r.randint(0, 1 << 20, (len(sections), T))
    pos[:, 0] = (1 << 31) - 1 if T > 1 else 0
    q, k = (to_type(r.randn(T, n, D), t) for n in (H, KV))
    src = [View(qm, a, t, layout) for a in (q, k)]
    dst = [View(qm, np.zeros_like(a), t, layout, fill=7) for a in (q, k)]
    R = qm.Rope.make(D, rot, sections, turns, adjacent, theta)
    p = ints(qm, pos)
    both = lambda vs: (qm.Heads * 2)(vs[0].heads[0], vs[1].heads[0])  # noqa: E731
    qm.rope_dev(R, p.ptr, T, t, both(src), both(dst))
    for a, s, d in zip((q, k), src, dst):
        x = values(a, t)
        want = rope(x, pos, rot, sections, turns, adjacent, theta)
        got, rest = d.read()
        assert rest
        got = values(got, t)
        # at position 2^31 the two sides' frequencies (2^-52 each) and 64-bit products (2^-53 each) put
        # their angles up to 2 (2^-21 + 2^-22) apart, the fraction of a turn in fp32 2 pi 2^-26 more:
        # under 2^-19; cosine and sine are off by 2 steps of 2^-24, a product and a sum of two round
        # three times; then the type's own half step
        i, j = np.arange(D), np.arange(D)
        half = rot // 2
        j = np.where(i >= rot, i, i ^ 1 if adjacent else np.where(i < half, i + half, i - half))
        tol = np.where(i < rot, (np.abs(x) + np.abs(x[..., j])) * (2.0 ** -19 + 5 * 2.0 ** -24), 0.0)
        close(got, want, tol + HALF[t] * np.abs(want) + 2.0 ** -25 * (t == F16), "rope")
        assert np.array_equal(got[..., rot:], x[..., rot:])
        # in place
        qm.rope_dev(R, p.ptr, T, t, s.heads, s.heads)
        again, rest = s.read()
        assert rest and np.array_equal(again, d.read()[0])


def test_rope_fused_projection_in_place(qm):
    """q and k in one buffer, side by side in a token, and q beside a gate within a head."""
    T, H, KV, D = 6, 4, 2, 64
    r = rng_of(1, 2)
    x = r.randn(T, (H * 2 + KV) * D).astype(np.float32)
    buf = qm.DBuf.from_array(x)
    row = x.shape[1]
    hs = qm.heads((buf.ptr, H, row, 2 * D), (buf.ptr + 4 * 2 * H * D, KV, row, D))
    pos = r.randint(0, 5000, (3, T))
    qm.rope_dev(qm.Rope.make(D, 32, (6, 5, 5), True, False, 1e7), ints(qm, pos).ptr, T, F32, hs, hs)
    got = buf.download(np.float32).reshape(x.shape)
    q = x[:, :2 * H * D].reshape(T, H, 2, D)
    want = rope(q[:, :, 0].astype(np.float64), pos, 32, (6, 5, 5), True, False, 1e7)
    gq = got[:, :2 * H * D].reshape(T, H, 2, D)
    # angles of a few thousand: 2 pi 2^-26 and five roundings of 2^-24 of two values of up to 5
    close(gq[:, :, 0], want, 10 * (2 * np.pi * 2.0 ** -26 + 5 * 2.0 ** -24))
    assert np.array_equal(gq[:, :, 1], q[:, :, 1])
    k = x[:, 2 * H * D:].reshape(T, KV, D).astype(np.float64)
    close(got[:, 2 * H * D:].reshape(T, KV, D), rope(k, pos, 32, (6, 5, 5), True, False, 1e7),
          10 * (2 * np.pi * 2.0 ** -26 + 5 * 2.0 ** -24))


# -------------------------------------------------------------- bookkeeping --

class Pool:
    def __init__(self, qm, n_seq, max_blocks, bs, n_block, table, free):
        self.table, self.free = ints(qm, table), ints(qm, free)
        self.c = qm.KvTable(n_seq, max_blocks, bs, n_block, self.table.ptr, self.free.ptr)
        self.n_block, self.shape = n_block, (n_seq, max_blocks)

    def read(self):
        n = self.shape[0] * self.shape[1]
        return self.table.download(np.int32, n).reshape(self.shape), self.free.download(np.int32, self.n_block)


def assign_ref(table, free, top, held_, new, bs, T, max_blocks, n_block):
    """(status, table, slot, pos, cu, len, n_free)"""
    slot, pos = np.full(T, -1), np.zeros(T, int)
    fail = lambda st: (st, table, slot, pos, np.zeros(len(held_) + 1, int), held_, top)  # noqa: E731
    if (np.minimum(held_, new) < 0).any() or new.sum() > T:
        return fail(3)
    after, had = -(-(held_ + new) // bs), -(-held_ // bs)
    if (after > max_blocks).any():
        return fail(2)
    if not 0 <= top <= n_block:
        return fail(4)
    if (after - had).sum() > top:
        return fail(1)
    table, at = table.copy(), 0
    cu = [0]
    for i in range(len(held_)):
        for c in range(had[i], after[i]):
            top -= 1
            table[i, c] = free[top]
        for j in range(new[i]):
            p = held_[i] + j
            slot[at], pos[at] = table[i, p // bs] * bs + p % bs, p
            at += 1
        cu.append(at)
    return 0, table, slot, pos, np.array(cu), held_ + new, top


def run_assign(qm, pool, held_, new, top, T, shift=0):
    n = pool.shape[0]
    out = {k: qm.DBuf.from_array(np.full(max(1, size) + 4, 77, np.int32))
           for k, size in (("slot", T), ("pos", T), ("cu", n + 1), ("len", n), ("n_free", 1), ("status", 1))}
    at = {k: b.ptr + 4 * shift for k, b in out.items()}
    a, b, c = ints(qm, held_), ints(qm, new), ints(qm, [top])
    qm.kv_assign_dev(pool.c, a.ptr, b.ptr, c.ptr, T, at["slot"], at["pos"], at["cu"], at["len"], at["n_free"], at["status"])
    got = {k: b.download(np.int32)[shift:] for k, b in out.items()}
    for k, size in (("slot", T), ("pos", T), ("cu", n + 1), ("len", n), ("n_free", 1), ("status", 1)):
        assert (got[k][size:] == 77).all(), k            # nothing behind the end
        got[k] = got[k][:size]
    return got


@pytest.mark.parametrize("n_seq,T,most,bs,shift", [(1, 1, 1, 16, 0), (3, 40, 12, 16, 0), (48, 48, 1, 32, 1), (70, 5000, 200, 64, 0),
                                                   (300, 3000, 9, 128, 2), (4096, 4096, 1, 16, 0), (513, 33333, 130, 256, 3),
                                                   (5, 0, 0, 16, 0), (0, 4, 0, 16, 0)])
def test_assign_and_release(qm, n_seq, T, most, bs, shift):
    r = rng_of(n_seq, T, bs)
    max_blocks = 40
    held_ = r.randint(0, 20 * bs, n_seq)
    held_[: n_seq // 3] = bs * (held_[: n_seq // 3] // bs)           # on a block's border
    new = np.zeros(n_seq, int)
    for i in r.permutation(n_seq):
        new[i] = min(r.randint(0, most + 1), T - new.sum())
    used = -(-held_ // bs)
    n_block = int(used.sum() + (-(-(held_ + new) // bs) - used).sum()) + 2
    order = r.permutation(n_block)
    table = np.full((n_seq, max_blocks), -1)
    table[np.arange(max_blocks)[None] < used[:, None]] = order[:used.sum()]
    free = np.full(n_block, -5)
    top = n_block - int(used.sum())
    free[:top] = order[used.sum():]
    pool = Pool(qm, n_seq, max_blocks, bs, n_block, table, free)
    want = assign_ref(table, free, top, held_, new, bs, T, max_blocks, n_block)
    for _ in range(2):                                                # issued again: the same
        got = run_assign(qm, pool, held_, new, top, T, shift)
        assert got["status"][0] == want[0] == 0
        t, f = pool.read()
        assert np.array_equal(t, want[1]) and np.array_equal(f, free)
        for k, w in zip(("slot", "pos", "cu", "len"), want[2:6]):
            assert np.array_equal(got[k], w), k
        assert got["n_free"][0] == want[6]
    # some sequences end
    ended = (r.rand(n_seq) < 0.4).astype(int) * 3
    length, n_free = want[5], want[6]
    ln, nf, st = (qm.DBuf.from_array(np.full(max(1, n), 77, np.int32)) for n in (n_seq, 1, 1))
    a, b, c = ints(qm, length), ints(qm, ended), ints(qm, [n_free])
    for _ in range(2):
        qm.kv_release_dev(pool.c, a.ptr, b.ptr, c.ptr, ln.ptr, nf.ptr, st.ptr)
        back = [x for i in range(n_seq) if ended[i] for x in want[1][i, :-(-length[i] // bs)]]
        t, f = pool.read()
        assert st.download(np.int32)[0] == 0 and nf.download(np.int32)[0] == n_free + len(back)
        assert np.array_equal(t, want[1])
        assert np.array_equal(f[n_free:n_free + len(back)], back) and np.array_equal(f[:n_free], free[:n_free])
        if n_seq:
            assert np.array_equal(ln.download(np.int32, n_seq), np.where(ended, 0, length))


@pytest.mark.parametrize("why,status", [("full", 1), ("row", 2), ("negative", 3), ("negative new", 3), ("too many", 3),
                                        ("overflow", 3), ("list", 4), ("list negative", 4)])
def test_assign_refused_on_the_device(qm, why, status):
    """A step that cannot be served changes nothing and says why."""
    bs, max_blocks, n_block, T = 16, 4, 12, 100
    held_, new, top = np.array([10, 32, 0]), np.array([10, 20, 5]), 12
    table = np.arange(12).reshape(3, 4)
    free = np.arange(12)[::-1].copy()
    if why == "full":
        top = 3
    if why == "row":
        new[1] = 33
    if why == "negative":
        held_[2] = -1
    if why == "negative new":
        new[0] = -3
    if why == "too many":
        T = 34
    if why == "overflow":
        held_[0], new[0] = 2 ** 31 - 5, 10
    if why == "list":
        top = 13
    if why == "list negative":
        top = -1
    pool = Pool(qm, 3, max_blocks, bs, n_block, table, free)
    got = run_assign(qm, pool, held_, new, top, T)
    assert got["status"][0] == status
    t, f = pool.read()
    assert np.array_equal(t, table) and np.array_equal(f, free)
    assert (got["slot"] == -1).all() and (got["pos"] == 0).all() and (got["cu"] == 0).all()
    assert np.array_equal(got["len"], held_) and got["n_free"][0] == top


def test_release_refused_on_the_device(qm):
    table, free = np.arange(12).reshape(3, 4), np.arange(12)
    pool = Pool(qm, 3, 4, 16, 12, table, free)
    for held_, top, status in (([64, 64, 1], 6, 4), ([65, 0, 0], 0, 2), ([-1, 0, 0], 0, 3), ([1, 1, 1], 13, 4)):
        a, b, c = ints(qm, held_), ints(qm, [1, 1, 0]), ints(qm, [top])
        ln, nf, st = ints(qm, [9, 9, 9]), ints(qm, [9]), ints(qm, [9])
        qm.kv_release_dev(pool.c, a.ptr, b.ptr, c.ptr, ln.ptr, nf.ptr, st.ptr)
        assert st.download(np.int32)[0] == status and nf.download(np.int32)[0] == top
        assert np.array_equal(ln.download(np.int32), held_)
        assert np.array_equal(pool.read()[1], free)


# ------------------------------------------------------------------- cache --

def kv_values(r, shape):
    x = r.randn(*shape) * np.exp(r.randn(*shape[-2:]) * 0.7) + r.randn(*shape[-2:])
    return x


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("T,KV,D,bs,layout", [(1, 2, 256, 16, "packed"), (7, 2, 256, 32, "gap"), (50, 8, 128, 64, "odd"),
                                              (129, 3, 64, 16, "heads"), (1000, 1, 128, 256, "packed")])
def test_append_and_read(qm, typ, T, KV, D, bs, layout):
    t = TYPES[typ]
    r = rng_of(T, KV, D)
    n_block = T // bs + 3
    k, v = (kv_values(r, (T, KV, D)) for _ in range(2))
    k[0, 0, :64] = 2.5                                   # one value: no step
    v[-1, -1, :64] = np.arange(64) / 8.0                 # codes on a border
    k[T // 2, 0, -64:] *= 1e-6                           # steps below fp16's normal range
    k, v = to_type(k, t), to_type(v, t)
    slot = r.permutation(n_block * bs)[:T]
    if T > 2:
        slot[1], slot[2] = -1, n_block * bs              # outside: left out
    data = r.randint(0, 256, (n_block, KV, bs * (D + D // 8))).astype(np.uint8)
    cache = qm.DBuf.from_array(data)
    c = qm.Kv4(cache.ptr, n_block, bs, KV, D)
    assert qm.kv4_block_bytes(c) == data[0].size
    kv_, vv_ = View(qm, k, t, layout), View(qm, v, t, layout)
    sl = ints(qm, slot)
    qm.kv4_append_dev(c, t, kv_.heads, vv_.heads, sl.ptr, T)
    # the bytes, by the layout's own formulas
    full_k, full_v = (np.zeros((n_block, KV, bs, D), np.float32) for _ in range(2))
    live = (slot >= 0) & (slot < n_block * bs)
    for x, full in ((k, full_k), (v, full_v)):
        full[slot[live] // bs, :, slot[live] % bs] = values(x, t)[live]
    want = block_bytes(full_k, full_v, bs)
    mask = block_bytes_mask(n_block, KV, bs, D, slot[live])
    got = cache.download(np.uint8).reshape(data.shape)
    assert np.array_equal(got[mask], want[mask])
    assert np.array_equal(got[~mask], data[~mask])       # other slots as they were
    ask = ints(qm, np.concatenate([slot, [-1]]))
    ko, vo = (qm.DBuf.from_array(np.full((T + 1) * KV * D, 7, np.float32)) for _ in range(2))
    qm.kv4_read_dev(c, ask.ptr, T + 1, ko.ptr, vo.ptr)
    for x, o in ((k, ko), (v, vo)):
        y = held(values(x, t).astype(np.float32)) * live[:, None, None]
        o = o.download(np.float32).reshape(T + 1, KV, D)
        assert np.array_equal(o[:T].astype(np.float64), y) and (o[T] == 0).all()


def block_bytes_mask(n_block, KV, bs, D, slots):
    """Bytes of the slots' tokens."""
    m = np.zeros((n_block, KV, bs * (D + D // 8)), bool)
    half = bs * (D // 2 + D // 16)
    for s in slots:
        b, o = s // bs, s % bs
        for base in (0, half):
            m[b, :, base + o * D // 2:base + (o + 1) * D // 2] = True
            at = base + bs * D // 2 + o * (D // 16)
            m[b, :, at:at + D // 16] = True
    return m


@pytest.mark.parametrize("typ", TYPES)
def test_append_of_what_fp16_does_not_hold(qm, typ):
    """Values beyond fp16's range saturate; a group with an infinity or a NaN is NaN."""
    t = TYPES[typ]
    D, bs = 128, 16
    x = np.zeros((6, 1, D), np.float32)
    x[:] = np.linspace(-1, 1, D)
    x[0, 0, 3] = np.nan
    x[1, 0, 70] = np.inf
    x[2, 0, 5] = -np.inf
    if t != F16:
        x[3, 0, 5] = -1e30
        x[4, 0, 64:] = 3e38
        x[4, 0, 70] = -3e38
    x = to_type(x, t)
    cache = qm.DBuf(bs * (D + D // 8))
    c = qm.Kv4(cache.ptr, 1, bs, 1, D)
    view, sl = View(qm, x, t), ints(qm, np.arange(6))
    qm.kv4_append_dev(c, t, view.heads, view.heads, sl.ptr, 6)
    ko, vo = qm.DBuf(4 * 6 * D), qm.DBuf(4 * 6 * D)
    qm.kv4_read_dev(c, sl.ptr, 6, ko.ptr, vo.ptr)
    want = held(values(x, t).astype(np.float32))
    for o in (ko, vo):
        got = o.download(np.float32).reshape(6, 1, D)
        assert np.array_equal(got.astype(np.float64), want, equal_nan=True)
    assert np.isnan(want[0, 0, :64]).all() and np.isfinite(want[0, 0, 64:]).all() and np.isnan(want[1, 0, 64:]).all()


# --------------------------------------------------- attention over the cache --

class CacheCase:
    """Sequences in a shuffled paged cache, with their float64 values."""

    def __init__(self, qm, r, lens, KV, D, bs, k=None, v=None, spare=2, extra_cols=1, junk=True):
        self.lens, self.bs, self.KV, self.D = np.asarray(lens), bs, KV, D
        used = -(-self.lens // bs)
        self.n_block = int(used.sum()) + spare
        order = r.permutation(self.n_block)
        cols = int(max(1, used.max() if len(used) else 1)) + extra_cols
        self.table = np.full((len(self.lens), cols), -1)
        at, kb, vb = 0, np.zeros((self.n_block, KV, bs, D), np.float32), np.zeros((self.n_block, KV, bs, D), np.float32)
        self.k, self.v = [], []
        for i, n in enumerate(self.lens):
            self.table[i, :used[i]] = order[at:at + used[i]]
            at += used[i]
            ki = kv_values(r, (n, KV, D)).astype(np.float32) if k is None else k[i]
            vi = r.randn(n, KV, D).astype(np.float32) if v is None else v[i]
            tok = np.arange(n)
            kb[self.table[i, tok // bs], :, tok % bs] = ki
            vb[self.table[i, tok // bs], :, tok % bs] = vi
            self.k.append(held(ki))
            self.v.append(held(vi))
        bytes_ = block_bytes_fast(kb, vb, bs)
        if junk:        # what lies behind the sequences' ends: anything, NaN among it
            m = np.ones(bytes_.shape, bool)
            for i, n in enumerate(self.lens):
                tok = np.arange(n)
                m &= ~block_bytes_mask_fast(self.n_block, KV, bs, D, self.table[i, tok // bs] * bs + tok % bs)
            bytes_[m] = 0xFF
        self.data = qm.DBuf.from_array(bytes_)
        self.table_dev = ints(qm, self.table)
        self.c = qm.Kv4(self.data.ptr, self.n_block, bs, KV, D)
        self.t = qm.KvTable(len(self.lens), cols, bs, self.n_block, self.table_dev.ptr, None)


def block_bytes_fast(k, v, bs):
    nb, kv, _, D = k.shape
    out = np.zeros((nb, kv, bs * (D + D // 8)), np.uint8)
    half, ng = bs * (D // 2 + D // 16), D // 64
    for x, base, is_k in ((k, 0, True), (v, half, False)):
        c, d, m = quantise(x)
        if is_k:
            c = c.reshape(nb, kv, bs, ng, 2, 4, 4, 2).transpose(0, 1, 2, 5, 3, 4, 6, 7)
        else:
            c = c.reshape(nb, kv, bs, ng, 16, 2, 2).transpose(0, 1, 2, 4, 3, 5, 6)
        c = c.reshape(nb, kv, bs * D // 2, 2)
        out[:, :, base:base + bs * D // 2] = c[..., 0] | (c[..., 1] << 4)
        out[:, :, base + bs * D // 2:base + half] = np.stack([d, m], -1).astype(np.float16).reshape(nb, kv, -1).view(np.uint8)
    return out


def block_bytes_mask_fast(n_block, KV, bs, D, slots):
    m = np.zeros((n_block, KV, bs * (D + D // 8)), bool)
    half = bs * (D // 2 + D // 16)
    tok = np.zeros((n_block, bs), bool)
    tok[np.asarray(slots, int) // bs, np.asarray(slots, int) % bs] = True
    for base in (0, half):
        m[:, :, base:base + bs * D // 2] |= np.repeat(tok, D // 2, 1)[:, None]
        m[:, :, base + bs * D // 2:base + half] |= np.repeat(tok, D // 16, 1)[:, None]
    return m


def test_block_layouts_agree(qm):
    r = rng_of(5, 5)
    for D in (64, 128, 256):
        k, v = (r.randn(2, 2, 16, D).astype(np.float32) for _ in range(2))
        assert np.array_equal(block_bytes(k, v, 16), block_bytes_fast(k, v, 16))
        s = np.array([1, 17, 30])
        assert np.array_equal(block_bytes_mask(2, 2, 16, D, s), block_bytes_mask_fast(2, 2, 16, D, s))


def kv4_tol(t, D, L, want, mag, es):
    """es: max over keys of scale sum |q| |k|, with |k| <= 6 times what it is here (codes and minimum
    apart: d code and |m| are each at most the group's spread plus |k|, the spread at most 10 of |k|'s
    rms here).  fp32: q in two parts of 2^-22, sums of D products; weights in two parts, sums of L.
    16-bit: q exact, weights to 2^-11, the result to the type."""
    e = 6 * es * (2 ** -22 * (t == F32) + (D + 16) * 2.0 ** -24)
    w = 2.0 ** -21 if t == F32 else 2.0 ** -11
    return (2 * e + w + (L + 64) * 2.0 ** -24) * 6 * (mag + 0.5) + HALF[t] * np.abs(want)


def run_kv4(qm, case, q, ask, t, layout="packed", scale=None, pad=2, fill=5):
    T = int(np.sum(ask)) + pad
    H, D = q.shape[1], q.shape[2]
    cu = np.concatenate([[0], np.cumsum(ask)])
    qv = View(qm, q, t, layout)
    out = View(qm, np.full(q.shape, fill, q.dtype), t, layout, fill=fill)
    cu_d, len_d = ints(qm, cu), ints(qm, case.lens)
    scale = D ** -0.5 if scale is None else scale
    got = []
    for _ in range(2):
        qm.attn_kv4_dev(case.c, case.t, t, qv.heads, out.heads, cu_d.ptr, len_d.ptr, T, scale)
        y, rest = out.read()
        assert rest, "values between the rows"
        got.append(y)
    assert np.array_equal(got[0].view(np.uint8), got[1].view(np.uint8))      # equal calls, equal bits
    if pad:
        assert (got[0][cu[-1]:] == np.asarray(fill, q.dtype)).all()          # rows behind the last one
    return got[0][:cu[-1]]


def check_kv4(case, q, ask, t, got, scale=None):
    D = q.shape[2]
    at = 0
    for i, n in enumerate(ask):
        L = int(case.lens[i])
        qi = values(q[at:at + n], t)
        want, mag, es = attention(qi, case.k[i], case.v[i], L - n + np.arange(n), D ** -0.5 if scale is None else scale)
        close(values(got[at:at + n], t), want, kv4_tol(t, D, L, want, mag, es), (i, L, n))
        at += n


KV4_CASES = [
    # lens, rows that ask, heads, kv heads, D, block, layout
    ([1], [1], 2, 2, 64, 16, "packed"),
    ([33], [1], 8, 1, 128, 16, "packed"),
    ([700], [1], 16, 2, 256, 16, "gap"),
    ([2500], [1], 16, 2, 256, 64, "packed"),
    ([0, 5, 31, 32, 33, 300], [1, 1, 1, 1, 1, 1], 6, 2, 64, 32, "odd"),
    ([1200, 1, 17, 640, 16, 48], [1, 1, 1, 0, 1, 1], 12, 4, 128, 128, "packed"),
    ([100, 260], [3, 5], 4, 2, 128, 16, "heads"),
    ([90], [90], 4, 2, 64, 16, "packed"),
    ([515], [130], 8, 2, 256, 16, "packed"),
    ([300, 40, 0, 77], [64, 40, 3, 9], 3, 1, 128, 256, "odd"),
    ([3, 10], [5, 12], 4, 2, 64, 16, "packed"),            # more rows than tokens: the first see nothing
    ([64] * 70, [1] * 70, 2, 1, 64, 16, "packed"),
    ([40, 900], [1, 1], 34, 2, 64, 32, "packed"),          # 17 heads to a kv head
]


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("at", range(len(KV4_CASES)))
def test_attn_kv4(qm, typ, at):
    t = TYPES[typ]
    lens, ask, H, KV, D, bs, layout = KV4_CASES[at]
    r = rng_of(at, D)
    case = CacheCase(qm, r, lens, KV, D, bs)
    q = to_type(r.randn(sum(ask) + 2, H, D), t)
    got = run_kv4(qm, case, q, ask, t, layout)
    check_kv4(case, q, ask, t, got)


@pytest.mark.parametrize("typ", TYPES)
def test_attn_kv4_is_not_reached_by_what_it_does_not_see(qm, typ):
    """NaN, infinite and huge K and V of later tokens leave earlier rows alone; a row that sees
    them is not finite."""
    t = TYPES[typ]
    L, n, H, KV, D, bs = 70, 6, 4, 2, 128, 16
    r = rng_of(70, 6)
    k, v = kv_values(r, (L, KV, D)).astype(np.float32), r.randn(L, KV, D).astype(np.float32)
    q = to_type(r.randn(n, H, D), t)
    clean = CacheCase(qm, r, [L], KV, D, bs, [k], [v])
    want = run_kv4(qm, clean, q, [n], t, pad=0)
    for kind in ("nan", "inf", "huge"):
        k2, v2 = k.copy(), v.copy()
        bad = {"nan": np.nan, "inf": np.inf, "huge": 65000.0}[kind]
        k2[L - 3:, :, 5], v2[L - 3:, :, 70] = bad, bad
        dirty = CacheCase(qm, r, [L], KV, D, bs, [k2], [v2])
        got = run_kv4(qm, dirty, q, [n], t, pad=0)
        close(values(got[:n - 3], t), values(want[:n - 3], t),
              2 * kv4_tol(t, D, L, values(want[:n - 3], t), 3.0, 20.0), kind)
        if kind != "huge":
            assert not np.isfinite(values(got[n - 3:], t)).all()


def test_attn_kv4_bad_pages(qm):
    """A table entry outside the cache stands for tokens that are not there."""
    L, H, KV, D, bs = 100, 2, 1, 64, 16
    r = rng_of(3, 9)
    case = CacheCase(qm, r, [L, L], KV, D, bs)
    gone = np.zeros((2, L), bool)
    for i, c, bad in ((0, 1, -1), (0, 5, case.n_block), (1, 0, 2 ** 31 - 1), (1, 6, -2 ** 31)):
        case.table[i, c] = bad
        gone[i, c * bs:(c + 1) * bs] = True
    case.table_dev.upload(case.table.astype(np.int32))
    q = to_type(r.randn(2, H, D), F32)
    got = run_kv4(qm, case, q, [1, 1], F32, pad=0)
    for i in range(2):
        kk, vv = case.k[i][~gone[i]], case.v[i][~gone[i]]
        want, mag, es = attention(q[i:i + 1].astype(np.float64), kk, vv, [len(kk) - 1], D ** -0.5)
        close(got[i:i + 1], want, kv4_tol(F32, D, L, want, mag, es), i)
    case.table[:] = -1
    case.table_dev.upload(case.table.astype(np.int32))
    assert (run_kv4(qm, case, q, [1, 1], F32, pad=0) == 0).all()


@pytest.mark.parametrize("cu,lens", [([0, 9, 3], [20, 20]), ([-5, 2, 4], [20, 20]), ([0, 2, 1 << 30], [20, 20]),
                                     ([0, 2, 4], [-7, 1 << 30]), ([4, 0, 4], [20, 20])])
def test_attn_kv4_bad_lengths(qm, cu, lens):
    """Lengths that are none write no row outside the output (the results are not defined)."""
    r = rng_of(8, 1)
    case = CacheCase(qm, r, [20, 20], 1, 64, 16)
    q = View(qm, to_type(r.randn(4, 2, 64), F32), F32, "gap")
    out = View(qm, np.zeros((4, 2, 64), np.float32), F32, "gap", fill=3)
    qm.attn_kv4_dev(case.c, case.t, F32, q.heads, out.heads, ints(qm, cu).ptr, ints(qm, lens).ptr, 4, 0.125)
    assert out.read()[1]


# ------------------------------------------------------------------ prompts --

def prompt_tol(t, D, n, want, mag, es):
    """fp32: operands in two parts (2^-22 each, and the product of the low parts 2^-22), sums of D products and
    of n weights; 16-bit: operands exact, weights to the type's half step, the result too."""
    e = es * (3 * 2.0 ** -22 * (t == F32) + (D + 16) * 2.0 ** -24)
    w = 3 * 2.0 ** -22 if t == F32 else HALF[t]
    floor = n * 2.0 ** -25 * (t == F16)
    return (2 * e + w + (n + 64) * 2.0 ** -24) * mag + floor * (mag + 4) + HALF[t] * np.abs(want) + 1e-30


def run_prompt(qm, q, k, v, lens, t, layout="packed", scale=None, fill=5):
    T, H, D = q.shape
    cu = np.concatenate([[0], np.cumsum(lens)])
    views = [View(qm, a, t, layout) for a in (q, k, v)]
    out = View(qm, np.full(q.shape, fill, q.dtype), t, layout, fill=fill)
    c = ints(qm, cu)
    scale = D ** -0.5 if scale is None else scale
    got = []
    for _ in range(2):
        qm.attn_prompt_dev(t, D, *[x.heads for x in views], out.heads, c.ptr, len(lens), T, scale)
        y, rest = out.read()
        assert rest
        got.append(y)
    assert np.array_equal(got[0].view(np.uint8), got[1].view(np.uint8))
    assert (got[0][cu[-1]:] == np.asarray(fill, q.dtype)).all()
    return got[0]


def check_prompt(q, k, v, lens, t, got, scale=None, rows=None):
    D, at = q.shape[2], 0
    for i, n in enumerate(lens):
        js = np.arange(n) if rows is None else np.unique(np.clip(rows, 0, max(0, n - 1)))[:n]
        if n:
            want, mag, es = attention(values(q[at:at + n], t)[js], values(k[at:at + n], t), values(v[at:at + n], t), js,
                                      D ** -0.5 if scale is None else scale)
            close(values(got[at:at + n], t)[js], want, prompt_tol(t, D, n, want, mag, es), (i, n))
        at += n


PROMPT_CASES = [
    ([1], 0, 1, 1, 64, "packed"),
    ([5], 3, 2, 1, 128, "odd"),
    ([31, 32, 33], 0, 4, 2, 256, "packed"),
    ([0, 64, 0, 65, 1, 0], 2, 3, 3, 64, "gap"),
    ([127, 128, 129], 0, 2, 1, 128, "heads"),
    ([300], 1, 6, 2, 64, "packed"),
    ([270], 0, 4, 1, 256, "odd"),
    ([3] * 80, 0, 2, 2, 64, "packed"),
    ([200, 1, 150], 0, 5, 1, 128, "gap"),
]


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("at", range(len(PROMPT_CASES)))
def test_attn_prompt(qm, typ, at):
    t = TYPES[typ]
    lens, pad, H, KV, D, layout = PROMPT_CASES[at]
    r = rng_of(at, D, 3)
    T = sum(lens) + pad
    q, k, v = to_type(r.randn(T, H, D), t), to_type(kv_values(r, (T, KV, D)), t), to_type(r.randn(T, KV, D), t)
    got = run_prompt(qm, q, k, v, lens, t, layout)
    check_prompt(q, k, v, lens, t, got)


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attn_prompt_longer(qm, typ, D):
    """Several hundred tiles: a running maximum that moves, checked at a row of every workgroup."""
    t = TYPES[typ]
    r = rng_of(D, 11)
    lens = [1500, 700]
    T = sum(lens)
    q, k, v = r.randn(T, 2, D), kv_values(r, (T, 1, D)), r.randn(T, 1, D)
    k *= np.linspace(0.2, 2.0, T)[:, None, None]          # later keys outweigh earlier ones
    q, k, v = to_type(q, t), to_type(k, t), to_type(v, t)
    got = run_prompt(qm, q, k, v, lens, t)
    check_prompt(q, k, v, lens, t, got, rows=np.arange(0, 1500, 37))


@pytest.mark.parametrize("typ", TYPES)
def test_attn_prompt_is_not_reached_by_what_it_does_not_see(qm, typ):
    """NaN, infinite and huge keys and values of later tokens, of other prompts and behind the last one."""
    t = TYPES[typ]
    H, KV, D, lens = 2, 1, 64, [50, 40]
    T, at = 93, 20
    r = rng_of(17, 4)
    q, k, v = r.randn(T, H, D), kv_values(r, (T, KV, D)), r.randn(T, KV, D)
    big = {F32: 3e38, BF16: 3e38, F16: 65504.0}[t]
    a = [to_type(x, t) for x in (q, k, v)]
    want = values(run_prompt(qm, *a, lens, t), t)
    for bad in (np.nan, np.inf, -np.inf, big, -big):
        kb, vb = k.copy(), v.copy()
        kb[at, 0, 3], kb[90:] = bad, bad
        vb[at, 0, 7], vb[90:] = bad, bad
        b = [to_type(x, t) for x in (q, kb, vb)]
        got = values(run_prompt(qm, *b, lens, t), t)
        seen = (np.arange(T) >= at) & (np.arange(T) < 50)
        live = ~seen & (np.arange(T) < 90)
        assert np.array_equal(got[live], want[live]), bad
        if not np.isfinite(bad):
            assert not np.isfinite(got[seen]).all()


@pytest.mark.parametrize("typ", TYPES)
def test_attn_prompt_infinite_values(qm, typ):
    """V's infinities come through with their sign, and meet as NaN."""
    t = TYPES[typ]
    H, KV, D, n = 1, 1, 64, 40
    r = rng_of(23)
    q, k, v = 0.1 * r.randn(n, H, D), 0.1 * r.randn(n, KV, D), r.randn(n, KV, D)
    v[5, 0, 2], v[9, 0, 2], v[30, 0, 4], v[33, 0, 6] = np.inf, -np.inf, -np.inf, np.nan
    a = [to_type(x, t) for x in (q, k, v)]
    got = values(run_prompt(qm, *a, [n], t), t)[:, 0]
    assert np.isfinite(got[:5]).all() and np.isposinf(got[5:9, 2]).all() and np.isnan(got[9:, 2]).all()
    assert np.isfinite(got[:30, 4]).all() and np.isneginf(got[30:, 4]).all()
    assert np.isfinite(got[:33, 6]).all() and np.isnan(got[33:, 6]).all()
    other = np.setdiff1d(np.arange(D), [2, 4, 6])
    v[~np.isfinite(v)] = 0
    a[2] = to_type(v, t)
    plain = values(run_prompt(qm, *a, [n], t), t)[:, 0]
    assert np.array_equal(got[:, other], plain[:, other])


@pytest.mark.parametrize("typ", ["f32"])
@pytest.mark.parametrize("power", [-60, -20, 20, 40])
def test_attn_prompt_f32_range(qm, typ, power):
    """fp32 operands of any size: scaled by powers of two, the results scale with them bit for bit."""
    t = TYPES[typ]
    r = rng_of(31, 2)
    n, H, KV, D = 150, 2, 1, 128
    q, k, v = (r.randn(n, x, D).astype(np.float32) for x in (H, KV, KV))
    base = run_prompt(qm, q, k, v, [n], t)
    f = np.float32(2.0 ** power)
    got = run_prompt(qm, q * f, k / f, v * f, [n], t)
    assert np.array_equal(got, base * f)


@pytest.mark.parametrize("cu", [[0, 9, 3], [-5, 2, 4], [0, 2, 1 << 30], [4, 0, 4], [0, 40, 40]])
def test_attn_prompt_bad_lengths(qm, cu):
    """Lengths that are none write no row outside the output (the results are not defined)."""
    r = rng_of(8, 2)
    q, k, v = (View(qm, r.randn(40, n, 64).astype(np.float32), F32, "gap") for n in (2, 1, 1))
    out = View(qm, np.zeros((40, 2, 64), np.float32), F32, "gap", fill=3)
    qm.attn_prompt_dev(F32, 64, q.heads, k.heads, v.heads, out.heads, ints(qm, cu).ptr, 2, 40, 0.125)
    assert out.read()[1]


# ----------------------------------------------------------------- together --

def test_a_session(qm):
    """Two prompts, then decoded tokens, as a program runs them: blocks and slots, rotary positions
    on the projections' output, attention of the prompt, the cache filled, attention over it; one
    sequence ends and its blocks go to a third."""
    H, KV, D, bs, rot, sections, theta = 4, 2, 128, 16, 64, (12, 10, 10), 1e6
    n_seq, cols, n_block = 3, 8, 9
    r = rng_of(2, 7)
    R = qm.Rope.make(D, rot, sections, True, False, theta)
    pool = Pool(qm, n_seq, cols, bs, n_block, np.full((n_seq, cols), -1), np.arange(n_block))
    data = qm.DBuf.from_array(np.full(n_block * KV * bs * (D + D // 8), 0xFF, np.uint8))
    cache = qm.Kv4(data.ptr, n_block, bs, KV, D)
    lens, nfree = [ints(qm, np.zeros(n_seq)) for _ in range(2)], [ints(qm, [n_block]) for _ in range(2)]
    status = ints(qm, [9])
    hist = [[np.zeros((0, KV, D))] * 2 for _ in range(n_seq)]
    scale = D ** -0.5
    which = 0

    def step(new, prompt):
        nonlocal which
        T = int(sum(new))
        slot, pos, cu = (ints(qm, np.zeros(max(1, n))) for n in (T, T, n_seq + 1))
        n_new = ints(qm, new)
        qm.kv_assign_dev(pool.c, lens[which].ptr, n_new.ptr, nfree[which].ptr, T, slot.ptr, pos.ptr, cu.ptr,
                         lens[1 - which].ptr, nfree[1 - which].ptr, status.ptr)
        which = 1 - which
        assert status.download(np.int32)[0] == 0
        # q beside its gate, as the projection leaves it; one position for all three axes
        qg = r.randn(T, H, 2, D).astype(np.float32)
        k, v = kv_values(r, (T, KV, D)).astype(np.float32), r.randn(T, KV, D).astype(np.float32)
        qd, kd, vd = (qm.DBuf.from_array(x) for x in (qg, k, v))
        p = pos.download(np.int32, T)
        pos3 = ints(qm, np.stack([p] * 3))
        qk = qm.heads((qd.ptr, H, 2 * H * D, 2 * D), (kd.ptr, KV, KV * D, D))
        hv, out = qm.heads((vd.ptr, KV, KV * D, D)), qm.DBuf(4 * T * H * D)
        ho = qm.heads((out.ptr, H, H * D, D))
        hq, hk = (qm.Heads * 1)(qk[0]), (qm.Heads * 1)(qk[1])
        qm.rope_dev(R, pos3.ptr, T, F32, qk, qk)
        qm.kv4_append_dev(cache, F32, hk, hv, slot.ptr, T)
        if prompt:
            qm.attn_prompt_dev(F32, D, hq, hk, hv, ho, cu.ptr, n_seq, T, scale)
        else:
            qm.attn_kv4_dev(cache, pool.c, F32, hq, ho, cu.ptr, lens[which].ptr, T, scale)
        got = out.download(np.float32).reshape(T, H, D)
        kr = kd.download(np.float32).reshape(T, KV, D)                # the turned keys themselves: their codes are exact
        want_q = rope(qg[:, :, 0].astype(np.float64), np.stack([p] * 3), rot, sections, True, False, theta)
        close(kr, rope(k.astype(np.float64), np.stack([p] * 3), rot, sections, True, False, theta),
              2 * np.abs(k).max() * (2 * np.pi * 2.0 ** -26 + 5 * 2.0 ** -24))
        at = 0
        for i, n in enumerate(new):
            mine = slice(at, at + n)
            old = hist[i][0].shape[0]
            hist[i] = [np.concatenate([hist[i][j], held(x[mine])]) for j, x in enumerate((kr, v))]
            kk, vv = (kr[mine].astype(np.float64), v[mine].astype(np.float64)) if prompt else hist[i]
            if n:
                want, mag, es = attention(want_q[mine], kk, vv, (0 if prompt else old) + np.arange(n), scale)
                # the rotary error of q, 2^-21 of it, enters the scores
                close(got[mine], want, kv4_tol(F32, D, kk.shape[0], want, mag, es) + 8 * es * 2.0 ** -21 * (mag + 0.5), (i, n))
            at += n
        assert np.array_equal(lens[which].download(np.int32, n_seq), [x[0].shape[0] for x in hist])

    step([37, 20, 0], True)
    for _ in range(3):
        step([1, 1, 0], False)
    step([2, 12, 0], False)
    ended = ints(qm, [1, 0, 0])
    qm.kv_release_dev(pool.c, lens[which].ptr, ended.ptr, nfree[which].ptr, lens[1 - which].ptr, nfree[1 - which].ptr,
                      status.ptr)
    which = 1 - which
    hist[0] = [np.zeros((0, KV, D))] * 2
    step([0, 0, 70], True)                                             # needs the blocks given back
    step([0, 1, 1], False)
    assert nfree[which].download(np.int32, 1)[0] == n_block - 3 - 5
