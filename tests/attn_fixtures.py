"""What the attention tests share: the three activation types in numpy, heads
laid out in memory, plain 64-bit forms of the operators."""
import ctypes as C

import numpy as np

F32, F16, BF16 = 0, 1, 30
TYPES = {"f32": F32, "f16": F16, "bf16": BF16}
#: half a rounding step, relative
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def to_type(x, t):
    """x (float32 or float64) as stored values of the type: bytes in the array's own dtype."""
    x = np.asarray(x, dtype=np.float32)
    if t == F32:
        return x.copy()
    if t == F16:
        return x.astype(np.float16)
    u = x.view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def values(a, t):
    """float64 values of stored ones."""
    if t == BF16:
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def store_dtype(t):
    return {F32: np.float32, F16: np.float16, BF16: np.uint16}[t]


class View:
    """[T][H][D] stored values in one device buffer of a layout:
    packed; gap (wider strides of whole 16 bytes, odd places between); heads
    ([H][T][D]); odd (strides and start of no 16 bytes)."""

    def __init__(self, qm, a, t, layout="packed", fill=None):
        T, H, D = a.shape
        self.qm, self.t, self.shape = qm, t, a.shape
        if layout == "packed":
            start, ts, hs = 0, H * D, D
        elif layout == "gap":
            start, ts, hs = 16, H * (D + 16) + 32, D + 16
        elif layout == "heads":
            start, ts, hs = 0, D, T * D
        else:
            start, ts, hs = 3, H * (D + 1) + 5, D + 1
        self.start, self.ts, self.hs = start, ts, hs
        n = start + max(0, T - 1) * ts + (H - 1) * hs + D + 7
        self.host = np.full(n, 0, store_dtype(t)) if fill is None else np.full(n, fill, store_dtype(t))
        self.at = (start + np.arange(T)[:, None, None] * ts + np.arange(H)[None, :, None] * hs
                   + np.arange(D)[None, None, :])
        self.host[self.at] = a
        self.buf = qm.DBuf.from_array(self.host)
        self.heads = qm.heads((self.buf.ptr + start * self.host.itemsize, H, ts, hs))

    def read(self):
        """(values [T][H][D] as stored, whether everything between them is as it was)"""
        got = self.buf.download(self.host.dtype)
        rest = np.ones(got.size, bool)
        rest[self.at] = False
        same = np.array_equal(got[rest].view(np.uint8), self.host[rest].view(np.uint8))
        return got[self.at], same


def ints(qm, a):
    return qm.DBuf.from_array(np.asarray(a, dtype=np.int32).reshape(-1) if np.size(a) else np.zeros(1, np.int32))


# ------------------------------------------------------------------ oracle --

def rope_axes(sections, interleaved):
    left, axis, a = list(sections), [], 0
    while sum(left):
        while not left[a]:
            a = (a + 1) % len(left)
        axis.append(a)
        left[a] -= 1
        if interleaved:
            a = (a + 1) % len(left)
    return axis


def rope(x, pos, n_rot, sections, interleaved, adjacent, theta):
    """x [T][H][D] float64, pos [axes][T]."""
    i = np.arange(n_rot // 2)
    ang = np.asarray(pos, np.float64)[rope_axes(sections, interleaved)].T * theta ** (-2.0 * i / n_rot)
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    a, b = (2 * i, 2 * i + 1) if adjacent else (i, i + n_rot // 2)
    y = x.copy()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    return y


def attention(q, k, v, last, scale):
    """One sequence: q [n][H][D], k and v [L][KV][D] float64, row j sees tokens
    0 .. last[j].  Returns (out, weighted |v|, max_j sum |q||k| scale) for
    tolerances; a row that sees nothing is zero."""
    n, H, D = q.shape
    G = H // k.shape[1]
    out, mag, es = np.zeros((n, H, D)), np.zeros((n, H, D)), np.zeros((n, H, 1))
    for j in range(n):
        L = min(last[j] + 1, k.shape[0])
        if L <= 0:
            continue
        for h in range(H):
            kk, vv = k[:L, h // G], v[:L, h // G]
            s = kk @ q[j, h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[j, h], mag[j, h] = p @ vv, p @ np.abs(vv)
            es[j, h] = (np.abs(kk) @ np.abs(q[j, h])).max() * abs(scale)
    return out, mag, es


def quantise(x):
    """Codes, steps and minima of x [..., D] float32, the format's own fp32 steps."""
    x = np.asarray(x, np.float32)
    g = x.reshape(*x.shape[:-1], x.shape[-1] // 64, 64)
    with np.errstate(all="ignore"):
        lo, hi = g.min(-1), g.max(-1)
        d = np.minimum((hi - lo) * np.float32(1 / 15), np.float32(65504)).astype(np.float16)
        m = np.clip(lo, -65504, 65504).astype(np.float16)
        df = d.astype(np.float32)[..., None]
        c = np.where(df > 0, np.clip(np.rint((g - m.astype(np.float32)[..., None]) / df), 0, 15), 0)
    ok = np.isfinite(g).all(-1)
    d, m = np.where(ok, d, np.float16(np.nan)), np.where(ok, m, np.float16(0))
    return np.where(ok[..., None], c, 0).astype(np.uint8), d, m


def held(x):
    """float64 values the cache holds for x."""
    c, d, m = quantise(x)
    y = c.astype(np.float64) * d.astype(np.float64)[..., None] + m.astype(np.float64)[..., None]
    return y.reshape(np.shape(x)).astype(np.float32).astype(np.float64)


def block_bytes(k, v, block):
    """Block bytes of K, V [n_block][kv][block][D] float32, by the layout's formulas."""
    nb, kv, bs, D = k.shape
    out = np.zeros((nb, kv, bs * (D + D // 8)), np.uint8)
    ch = np.arange(D)
    g, r = ch // 64, ch % 64
    # (byte of a token's row, upper nibble) of each channel
    k_at = 4 * ((r % 32 // 8) * (D // 32) + 2 * g + r // 32) + (r % 8) // 2
    v_at = 2 * ((r // 4) * (D // 64) + g) + (r % 4) // 2
    half = bs * (D // 2 + D // 16)
    for x, at, base in ((k, k_at, 0), (v, v_at, half)):
        c, d, m = quantise(x)
        c = c.reshape(nb, kv, bs, D)
        for t in range(bs):
            for i in range(D):
                out[:, :, base + t * D // 2 + at[i]] |= c[:, :, t, i] << (4 * (i % 2))
        s = np.stack([d, m], -1).astype(np.float16)
        out[:, :, base + bs * D // 2:base + half] = s.reshape(nb, kv, -1).view(np.uint8)
    return out
