"""Performance cases of the attention entries: what a program that keeps a model's
attention on the device calls between the projections and the MoE layer.

  rope     qmag_rope_dev: rotary positions with one to four axes on q and k
  slots    qmag_kv_release_dev, qmag_kv_assign_dev: one scheduler step of a paged cache,
           ended sequences' blocks given back, the new tokens' blocks, slots and positions
  append   qmag_kv4_append_dev, qmag_kv4_read_dev: tokens' K and V into the 4-bit cache,
           and the values it holds for them
  kv4      qmag_attn_kv4_dev: attention of the newest tokens over the 4-bit cache
  prompt   qmag_attn_prompt_dev: causal attention over whole packed prompts

Activations are f32, as the projections leave them, or 16-bit.  A cache block holds, for
each kv head, `block` tokens: K codes, K scales, V codes, V scales; 64 values share a
scale d and a minimum m (fp16), a value is d * code + m with a code of 0 to 15.
"""
import math
import os
import sys
from types import SimpleNamespace

import numpy as np
import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (30, torch.bfloat16)}
GROUP = 64


def listed():
    return [
        # one decoded token of the engine's attention layer, far into a session: q lies beside
        # its gate in the projection's output, 64 of 256 values turn, three axes in turn
        dict(name="rope_t1", kind="rope", T=1, heads=16, kv=2, dim=256, rot=64, axes="11,11,10", turns=True,
             adjacent=False, theta=1e7, start=200000, gate=True, type="f32"),
        # a prompt of text and an image, the axes' pairs in runs, the whole head turned
        dict(name="rope_t4096", kind="rope", T=4096, heads=32, kv=8, dim=128, rot=128, axes="16,24,24", turns=False,
             adjacent=False, theta=1e6, start=0, gate=False, type="bf16"),
        # a decode step of a small batch: one token each, some sequences ended
        dict(name="slots_decode", kind="slots", n_seq=48, new=1, T=48, block=16, max_len=8192, ended=0.1, mix=1),
        # a step that admits many prompts at once
        dict(name="slots_prompt", kind="slots", n_seq=509, new=1024, T=262144, block=32, max_len=4096, ended=0.2, mix=2),
        # a few sequences' decoded tokens into the cache, the engine's kv heads
        dict(name="append_t7", kind="append", T=7, kv=2, dim=256, block=16, n_block=512, type="f32"),
        # a large prompt into the cache, an odd number of tokens
        dict(name="append_t16001", kind="append", T=16001, kv=8, dim=128, block=64, n_block=320, type="bf16"),
        # decode of one sequence with a long context, the engine's heads
        dict(name="kv4_t1_32k", kind="kv4", n_seq=1, max_len=32768, q=1, heads=16, kv=2, dim=256, block=16, mix=1,
             type="f32"),
        # decode of a batch whose contexts differ widely
        dict(name="kv4_batch", kind="kv4", n_seq=32, max_len=16384, q=1, heads=32, kv=8, dim=128, block=32, mix=2,
             type="bf16"),
        # a chunk of 512 prompt tokens behind an already cached part
        dict(name="kv4_chunk", kind="kv4", n_seq=1, max_len=12001, q=512, heads=16, kv=2, dim=256, block=16, mix=3,
             type="f32"),
        # three short prompts packed, the smallest call of a prompt
        dict(name="prompt_t77", kind="prompt", n_seq=3, T=77, pad=3, heads=16, kv=2, dim=256, mix=1, type="f32"),
        # prompts of different lengths packed into one call
        dict(name="prompt_t8192", kind="prompt", n_seq=5, T=8192, pad=0, heads=32, kv=8, dim=128, mix=2, type="bf16"),
        # one long prompt of the engine's heads in its own type
        dict(name="prompt_f32", kind="prompt", n_seq=1, T=4096, pad=0, heads=16, kv=2, dim=256, mix=3, type="f32"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


SHAPES = [(16, 2, 256), (16, 16, 256), (32, 8, 128), (32, 4, 128), (28, 4, 128), (40, 8, 64), (8, 8, 64), (6, 1, 128)]


def draw(rng):
    kind = rng.choice(["rope", "rope", "slots", "append", "kv4", "kv4", "kv4", "prompt", "prompt", "prompt"])
    heads, kv, dim = rng.choice(SHAPES)
    typ = rng.choice(["f32", "f32", "f16", "bf16"])
    mix = rng.randrange(1 << 30)
    if kind == "rope":
        rot = rng.choice([dim, dim // 2, dim // 4])
        axes = [rot // 2]
        while len(axes) < 4 and axes[0] > 4 and rng.random() < 0.7:
            n = rng.randint(1, axes[0] // 2)
            axes = [axes[0] - n] + axes[1:] + [n]
        return dict(kind="rope", T=_log_int(rng, 1, 2048 if typ == "f32" else 4096), heads=heads, kv=kv, dim=dim, rot=rot,
                    axes=",".join(str(a) for a in axes), turns=rng.random() < 0.5, adjacent=rng.random() < 0.5,
                    theta=rng.choice([1e4, 1e6, 1e7]), start=_log_int(rng, 1, 1000000), gate=rng.random() < 0.3, type=typ)
    if kind == "slots":
        n_seq, new = _log_int(rng, 1, 512), rng.choice([1, 1, _log_int(rng, 2, 1024)])
        return dict(kind="slots", n_seq=n_seq, new=new, T=n_seq * new if new == 1 else n_seq * (new // 2 + 1),
                    block=rng.choice([16, 32, 64, 128]), max_len=_log_int(rng, new, 8192), ended=rng.choice([0.0, 0.1, 0.3]),
                    mix=mix)
    if kind == "append":
        T, block = _log_int(rng, 1, 16384 * 1024 // (kv * dim * (2 if typ == "f32" else 1))), rng.choice([16, 32, 64, 128])
        return dict(kind="append", T=T, kv=kv, dim=dim, block=block, n_block=T // block + rng.randint(1, 64), type=typ)
    if kind == "kv4":
        n_seq = _log_int(rng, 1, 48)
        max_len = _log_int(rng, 1, min(32768, (1 << 29) // (n_seq * kv * dim)))
        q = 1 if rng.random() < 0.5 else min(max_len, _log_int(rng, 2, 512 if n_seq == 1 else 8), 6000000 // max_len)
        return dict(kind="kv4", n_seq=n_seq, max_len=max_len, q=q, heads=heads, kv=kv, dim=dim,
                    block=rng.choice([16, 32, 64, 128]), mix=mix, type=typ)
    n_seq = _log_int(rng, 1, 12)
    T = _log_int(rng, n_seq, 4096 if typ == "f32" or n_seq < 4 else 8192)
    return dict(kind="prompt", n_seq=n_seq, T=T, pad=rng.choice([0, 0, 5]), heads=heads, kv=kv, dim=dim, mix=mix, type=typ)


# ----------------------------------------------------------------- lengths --

def _prompt_lens(case):
    """Lengths of the packed prompts, T in all; of four or more one is empty."""
    r = np.random.RandomState(case["mix"] % (1 << 31))
    n, T = case["n_seq"], case["T"]
    live = n - 1 if n >= 4 else n
    cut = np.sort(r.choice(np.arange(1, T), live - 1, replace=False)) if live > 1 else np.zeros(0, np.int64)
    lens = np.diff(np.concatenate([[0], cut, [T]])).astype(np.int64)
    return np.insert(lens, r.randint(0, live + 1), 0) if live < n else lens


def _kv_lens(case):
    """(tokens in the cache, newest tokens that ask) of each sequence."""
    r = np.random.RandomState(case["mix"] % (1 << 31))
    n, top = case["n_seq"], case["max_len"]
    lens = np.exp(r.uniform(0, math.log(top), n)).round().astype(np.int64).clip(1, top)
    lens = np.maximum(lens, r.randint(1, top + 1, n) // 2).clip(1, top)
    lens[r.randint(0, n)] = top
    ask = np.ones(n, np.int64) if case["q"] == 1 else r.randint(1, case["q"] + 1, n)
    ask[int(np.argmax(lens))] = case["q"]
    return lens, np.minimum(ask, lens)


def _slot_lens(case):
    """(tokens held, new tokens, ended) of each sequence; the new ones fit T."""
    r = np.random.RandomState(case["mix"] % (1 << 31))
    n, top = case["n_seq"], case["max_len"]
    ended = r.rand(n) < case["ended"]
    new = np.ones(n, np.int64) if case["new"] == 1 else r.randint(0, case["new"] + 1, n)
    new[ended] = 0
    over = np.cumsum(new) - case["T"]
    new = np.where(over > 0, np.maximum(0, new - np.maximum(0, over)), new)
    held = np.minimum(r.randint(0, top + 1, n), np.maximum(0, top - new))
    held[ended] = np.maximum(1, held[ended])
    return held, new, ended


def _ceil(a, b):
    return -(-a // b)


# ------------------------------------------------------------------ inputs --

def _gen(seed, tag):
    g = torch.Generator(device=DEV)
    g.manual_seed((seed * 1000003 + tag * 7919 + 1) & 0x7FFFFFFFFFFFFFFF)
    return g


def _normal(seed, tag, shape, dtype=torch.float32):
    return torch.randn(shape, device=DEV, generator=_gen(seed, tag)).to(dtype)


def _keys(seed, tag, shape, dtype=torch.float32):
    """Keys: channels of different spread and mean, as a projection and its norm leave them."""
    g = _gen(seed, tag)
    spread = torch.exp(0.5 * torch.randn(shape[-2:], device=DEV, generator=g))
    mean = 0.5 * torch.randn(shape[-2:], device=DEV, generator=g)
    return (torch.randn(shape, device=DEV, generator=g) * spread + mean).to(dtype)


def _ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)


def _quantise(x):
    """Codes [..., D] (uint8), scale and minimum [..., D / 64] (fp16) of x (f32), the format's own fp32 steps."""
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    lo, hi = g.amin(-1), g.amax(-1)
    d = ((hi - lo) / 15.0).clamp(max=65504.0).half()
    m = lo.clamp(-65504.0, 65504.0).half()
    df = d.float().unsqueeze(-1)
    q = torch.where(df > 0, torch.round((g - m.float().unsqueeze(-1)) / df), torch.zeros_like(g)).clamp(0, 15)
    return q.to(torch.uint8).reshape(x.shape), d, m


def _pack(codes, d, m, is_k):
    """Block bytes of one tensor: codes and scales of [n_block, kv, block, ...]."""
    nb, kv, bs, D = codes.shape
    ng = D // GROUP
    if is_k:    # byte [h][g][s][b]: channels g * 64 + s * 32 + h * 8 + 2 b and the next
        c = codes.reshape(nb, kv, bs, ng, 2, 4, 4, 2).permute(0, 1, 2, 5, 3, 4, 6, 7)
    else:       # byte [i][g][b]: channels g * 64 + i * 4 + 2 b and the next
        c = codes.reshape(nb, kv, bs, ng, 16, 2, 2).permute(0, 1, 2, 4, 3, 5, 6)
    c = c.reshape(nb, kv, bs * D // 2, 2)
    s = torch.stack([d, m], -1).reshape(nb, kv, bs * ng * 2).view(torch.uint8)
    return torch.cat([c[..., 0] | (c[..., 1] << 4), s], -1)


def _cache(seed, n_block, kv, block, dim):
    """A filled cache [n_block, kv, bytes], some blocks at a time."""
    out = torch.empty((n_block, kv, block * (dim + dim // 8)), dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 26) // (kv * block * dim))
    for i, a in enumerate(range(0, n_block, step)):
        n = min(step, n_block - a)
        k = _keys(seed, 50 + 2 * i, (block, n, kv, dim)).permute(1, 2, 0, 3)
        v = _normal(seed, 51 + 2 * i, (n, kv, block, dim))
        out[a:a + n] = torch.cat([_pack(*_quantise(k), True), _pack(*_quantise(v), False)], -1)
    return out


def _positions(case):
    """Positions [axes, T]: text, then an image's grid that starts where the text ends."""
    T, n = case["T"], len(case["axes"].split(","))
    i = np.arange(T)
    text = _ceil(T, 2) if n > 1 else T
    side = max(1, int(math.sqrt(T - text)))
    j = np.maximum(i - text, 0)
    pos = np.stack([np.where(i < text, i, text + at) for at in (0 * j, j // side, j % side, j % 7)][:n])
    return case["start"] + pos


def _heads(t, n, dim, row=None):
    """How the library's calls take heads: rows of `row` values, a head every row / n values."""
    row = row or n * dim
    return (t.data_ptr(), n, row, row // n)


def _kv_step(case, seed):
    """Table, free list and lengths of a paged cache in use."""
    held, new, ended = _slot_lens(case)
    r = np.random.RandomState(seed % (1 << 31))
    at = r.permutation(case["n_seq"])
    held, new, ended = held[at], new[at], ended[at]
    bs = case["block"]
    used = _ceil(held, bs)
    width = _ceil(case["max_len"], bs) + 1
    n_block = int(used.sum() + _ceil(held + new, bs).sum() - used.sum()) + 16
    order = r.permutation(n_block).astype(np.int32)
    table = np.full((case["n_seq"], width), -1, np.int32)
    table[np.arange(width)[None] < used[:, None]] = order[:used.sum()]
    free = np.full(n_block, -1, np.int32)
    n_free = n_block - int(used.sum())
    free[:n_free] = order[used.sum():]
    return SimpleNamespace(held=held, new=new, ended=ended.astype(np.int32), table=table, free=free, n_free=n_free,
                           n_block=n_block)


def _append_slots(case, seed):
    r = np.random.RandomState(seed % (1 << 31))
    slot = r.permutation(case["n_block"] * case["block"])[:case["T"]]
    if case["T"] > 4:
        slot[r.randint(0, case["T"])] = -1      # a padded row of a batch
    return slot


def _kv_table(case, seed, lens):
    """Block table [n_seq, width] over a pool of blocks in any order; -1 behind a row's last block."""
    r = np.random.RandomState(seed % (1 << 31))
    used = _ceil(lens, case["block"])
    n_block = int(used.sum()) + 3
    width = int(used.max()) + 2
    table = np.full((case["n_seq"], width), -1, np.int32)
    table[np.arange(width)[None] < used[:, None]] = r.permutation(n_block)[:used.sum()]
    return table, n_block


def _inputs(case, seed):
    """Everything a call reads, on the GPU; lengths stand in numpy too."""
    k = case["kind"]
    s = SimpleNamespace(case=case)
    if k == "rope":
        dt, T, dim = TYPES[case["type"]][1], case["T"], case["dim"]
        s.pos = _ints(_positions(case))
        s.q = _normal(seed, 1, (T, case["heads"], dim * (2 if case["gate"] else 1)), dt)
        s.k = _keys(seed, 2, (T, case["kv"], dim), dt)
    elif k == "slots":
        s.step = _kv_step(case, seed)
        st = s.step
        s.held, s.new, s.ended, s.table, s.free = (_ints(x) for x in (st.held, st.new, st.ended, st.table, st.free))
        s.n_free = _ints([st.n_free])
    elif k == "append":
        dt = TYPES[case["type"]][1]
        s.k = _keys(seed, 1, (case["T"], case["kv"], case["dim"]), dt)
        s.v = _normal(seed, 2, (case["T"], case["kv"], case["dim"]), dt)
        s.slot = _ints(_append_slots(case, seed))
    elif k == "kv4":
        s.lens, s.ask = _kv_lens(case)
        s.cu = np.concatenate([[0], np.cumsum(s.ask)])
        s.T = int(s.cu[-1])
        table, s.n_block = _kv_table(case, seed, s.lens)
        s.width = table.shape[1]
        s.table, s.len_dev, s.cu_dev = _ints(table), _ints(s.lens), _ints(s.cu)
        s.cache = _cache(seed, s.n_block, case["kv"], case["block"], case["dim"])
        s.q = _normal(seed, 1, (s.T, case["heads"], case["dim"]), TYPES[case["type"]][1])
    else:
        dt, rows = TYPES[case["type"]][1], case["T"] + case["pad"]
        s.lens = _prompt_lens(case)
        s.cu = np.concatenate([[0], np.cumsum(s.lens)])
        s.rows, s.cu_dev = rows, _ints(s.cu)
        s.q = _normal(seed, 1, (rows, case["heads"], case["dim"]), dt)
        s.k = _keys(seed, 2, (rows, case["kv"], case["dim"]), dt)
        s.v = _normal(seed, 3, (rows, case["kv"], case["dim"]), dt)
    if "dim" in case:
        s.scale = 1.0 / math.sqrt(case["dim"])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    k = case["kind"]
    empty = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=DEV)  # noqa: E731
    if k == "rope":
        s.q_out = torch.empty((case["T"], case["heads"], case["dim"]), dtype=s.q.dtype, device=DEV)
        s.k_out = torch.empty_like(s.k)
        s.axis_sizes = [int(a) for a in case["axes"].split(",")]
        s.axis = _ints(_axis_of_pair(s.axis_sizes, case["turns"])).long()
    elif k == "slots":
        n = case["n_seq"]
        s.slot, s.pos, s.cu = empty(case["T"]), empty(case["T"]), empty(n + 1)
        s.len_mid, s.len_next, s.n_mid, s.n_next, s.status = empty(n), empty(n), empty(1), empty(1), empty(2)
        s.cols = torch.arange(s.table.shape[1], device=DEV)[None]
        s.rows = torch.arange(n, device=DEV)
    elif k == "append":
        s.cache = torch.zeros((case["n_block"], case["kv"], case["block"] * (case["dim"] + case["dim"] // 8)),
                              dtype=torch.uint8, device=DEV)
        s.k_out = torch.zeros((case["T"], case["kv"], case["dim"]), device=DEV)
        s.v_out = torch.zeros_like(s.k_out)
    else:
        s.out = torch.zeros_like(s.q)
    if own:
        _plan(s)
    torch.cuda.synchronize()            # the library works on a stream of its own
    return s


def _plan(s):
    """The descriptors that a program keeps beside its buffers."""
    sys.path.insert(0, os.path.join(os.getcwd(), "qwen-mobile-agent_amd"))
    import qmag
    qmag.init(0)
    s.lib, case = qmag, s.case
    k = case["kind"]
    if "type" in case:
        s.type = TYPES[case["type"]][0]
    if k == "rope":
        h, kv, d = case["heads"], case["kv"], case["dim"]
        s.rope = qmag.Rope.make(head_dim=d, n_rot=case["rot"], sections=s.axis_sizes, interleaved=case["turns"],
                                adjacent=case["adjacent"], theta=case["theta"])
        s.src = qmag.heads(_heads(s.q, h, d, s.q.shape[1] * s.q.shape[2]), _heads(s.k, kv, d))
        s.dst = qmag.heads(_heads(s.q_out, h, d), _heads(s.k_out, kv, d))
    elif k == "slots":
        s.pages = qmag.KvTable(case["n_seq"], s.table.shape[1], case["block"], s.step.n_block, s.table.data_ptr(),
                               s.free.data_ptr())
    elif k == "append":
        s.kv4 = qmag.Kv4(s.cache.data_ptr(), case["n_block"], case["block"], case["kv"], case["dim"])
        s.hk, s.hv = (qmag.heads(_heads(t, case["kv"], case["dim"])) for t in (s.k, s.v))
    elif k == "kv4":
        s.kv4 = qmag.Kv4(s.cache.data_ptr(), s.n_block, case["block"], case["kv"], case["dim"])
        s.pages = qmag.KvTable(case["n_seq"], s.width, case["block"], s.n_block, s.table.data_ptr(), None)
        s.hq, s.ho = (qmag.heads(_heads(t, case["heads"], case["dim"])) for t in (s.q, s.out))
    else:
        s.hq, s.ho = (qmag.heads(_heads(t, case["heads"], case["dim"])) for t in (s.q, s.out))
        s.hk, s.hv = (qmag.heads(_heads(t, case["kv"], case["dim"])) for t in (s.k, s.v))


def run(s):
    return {"rope": _run_rope, "slots": _run_slots, "append": _run_append, "kv4": _run_kv4,
            "prompt": _run_prompt}[s.case["kind"]](s)


# -------------------------------------------------------------------- rope --

def _axis_of_pair(sizes, turns):
    """The axis of each pair: its axes in runs, or in turns that pass over an axis with no pairs left."""
    if not turns:
        return np.repeat(np.arange(len(sizes)), sizes)
    n = max(sizes)
    turn = [(at, a) for a, size in enumerate(sizes) for at in range(size)]
    return np.array([a for at, a in sorted(turn)]) if n else np.zeros(0, np.int64)


def _turned(x, cos, sin, rot, adjacent):
    x = x.float()
    if adjacent:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _run_rope(s):
    case = s.case
    if own:
        s.lib.rope_dev(s.rope, s.pos.data_ptr(), case["T"], s.type, s.src, s.dst)
        return s.q_out, s.k_out
    rot = case["rot"]
    freq = torch.pow(case["theta"], torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / -rot)
    angle = s.pos[s.axis].double().T * freq         # far positions: 64 bits
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    q = s.q[..., :case["dim"]]
    return (_turned(q, cos, sin, rot, case["adjacent"]).to(s.q.dtype),
            _turned(s.k, cos, sin, rot, case["adjacent"]).to(s.k.dtype))


# ------------------------------------------------------------------- slots --

def _run_slots(s):
    case = s.case
    if own:
        s.lib.kv_release_dev(s.pages, s.held.data_ptr(), s.ended.data_ptr(), s.n_free.data_ptr(), s.len_mid.data_ptr(),
                             s.n_mid.data_ptr(), s.status.data_ptr())
        s.lib.kv_assign_dev(s.pages, s.len_mid.data_ptr(), s.new.data_ptr(), s.n_mid.data_ptr(), case["T"],
                            s.slot.data_ptr(), s.pos.data_ptr(), s.cu.data_ptr(), s.len_next.data_ptr(),
                            s.n_next.data_ptr(), s.status.data_ptr() + 4)
        return {"table": s.table, "free": s.free, "slot": s.slot, "pos": s.pos, "cu": s.cu, "len": s.len_next,
                "n_free": s.n_next, "status": s.status}
    bs, T = case["block"], case["T"]
    held, new, top = s.held.long(), s.new.long(), s.n_free.long()
    # ended sequences' blocks onto the free list, by sequence and column
    had = (held + bs - 1) // bs
    back = torch.where(s.ended > 0, had, torch.zeros_like(had))
    at = top + (torch.cumsum(back, 0) - back)[:, None] + s.cols
    given = s.cols < back[:, None]
    free = torch.cat([s.free, s.free.new_zeros(1)])         # one more place takes what is not given
    free.scatter_(0, torch.where(given, at, torch.full_like(at, s.free.numel())).flatten(), s.table.flatten())
    free, top = free[:-1], top + back.sum()
    held = torch.where(s.ended > 0, torch.zeros_like(held), held)
    # blocks of the new tokens from its end
    had, after = (held + bs - 1) // bs, held + new
    take = (after + bs - 1) // bs - had
    nth = (torch.cumsum(take, 0) - take)[:, None] + s.cols - had[:, None]
    taken = (s.cols >= had[:, None]) & (s.cols < (had + take)[:, None])
    fresh = free[(top - 1 - nth).clamp(0, free.numel() - 1)]
    table = torch.where(taken, fresh, s.table)
    cu = torch.cat([new.new_zeros(1), torch.cumsum(new, 0)])
    tok = torch.arange(T, device=DEV)
    row = torch.searchsorted(cu, tok, right=True) - 1
    live = row < case["n_seq"]
    row = row.clamp(max=case["n_seq"] - 1)
    pos = held[row] + tok - cu[row]
    slot = table[row, (pos // bs).clamp(0, table.shape[1] - 1)].long() * bs + pos % bs
    return {"table": table, "free": free, "slot": torch.where(live, slot, -1).int(),
            "pos": torch.where(live, pos, 0).int(), "cu": cu.int(), "len": after.int(),
            "n_free": (top - take.sum()).int().reshape(1), "status": torch.zeros_like(s.status)}


# ------------------------------------------------------------------ append --

def _held(x):
    """The f32 values the cache holds for x."""
    c, d, m = _quantise(x.float())
    g = c.float().reshape(*x.shape[:-1], -1, GROUP)
    return (g * d.float().unsqueeze(-1) + m.float().unsqueeze(-1)).reshape(x.shape)


def _run_append(s):
    case = s.case
    if own:
        s.lib.kv4_append_dev(s.kv4, s.type, s.hk, s.hv, s.slot.data_ptr(), case["T"])
        s.lib.kv4_read_dev(s.kv4, s.slot.data_ptr(), case["T"], s.k_out.data_ptr(), s.v_out.data_ptr())
        return s.k_out, s.v_out
    live = (s.slot >= 0)[:, None, None]
    return _held(s.k) * live, _held(s.v) * live


# --------------------------------------------------------------------- kv4 --

def _unpack(b, block, dim, is_k):
    """f32 values [..., block, dim] of block bytes."""
    ng, n = dim // GROUP, block * dim // 2
    c = torch.stack([b[..., :n] & 15, b[..., :n] >> 4], -1)
    lead = b.shape[:-1]
    if is_k:
        c = c.reshape(*lead, block, 4, ng, 2, 4, 2).movedim(-5, -3)
    else:
        c = c.reshape(*lead, block, 16, ng, 2, 2).transpose(-4, -3)
    c = c.reshape(*lead, block, ng, GROUP).float()
    dm = b[..., n:].contiguous().view(torch.float16).reshape(*lead, block, ng, 2).float()
    return (c * dm[..., 0:1] + dm[..., 1:2]).reshape(*lead, block, dim)


def _run_kv4(s):
    case = s.case
    if own:
        s.lib.attn_kv4_dev(s.kv4, s.pages, s.type, s.hq, s.ho, s.cu_dev.data_ptr(), s.len_dev.data_ptr(), s.T, s.scale)
        return s.out
    n, H, kv, D, bs = case["n_seq"], case["heads"], case["kv"], case["dim"], case["block"]
    G, Q = H // kv, case["q"]
    half = bs * (D // 2 + D // 16)
    pages = s.cache[s.table[:, :-2].long().clamp(min=0)]                # [n, blocks, kv, bytes]
    pages = pages.transpose(1, 2)
    K = _unpack(pages[..., :half], bs, D, True).reshape(n, kv, -1, D)   # [n, kv, L, D]
    V = _unpack(pages[..., half:], bs, D, False).reshape(n, kv, -1, D)
    L = K.shape[2]
    # queries padded to Q a sequence: [n, kv, Q * G, D]
    ask, start = (s.cu_dev[1:] - s.cu_dev[:-1]).long(), s.cu_dev[:-1].long()
    j = torch.arange(Q, device=DEV)[None]
    row = (start[:, None] + j).clamp(max=s.T - 1)
    q = s.q[row].float().reshape(n, Q, kv, G, D).transpose(1, 2).reshape(n, kv, Q * G, D)
    score = torch.matmul(q, K.transpose(2, 3).contiguous()).reshape(n, kv, Q, G, L) * s.scale
    last = s.len_dev.long()[:, None] - ask[:, None] + j                 # [n, Q]
    seen = torch.arange(L, device=DEV)[None, None] <= last[..., None]
    score = score.masked_fill(~seen[:, None, :, None], float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).reshape(n, kv, Q * G, L)
    o = torch.matmul(p, V).reshape(n, kv, Q, G, D).transpose(1, 2).reshape(n, Q, H, D)
    tok = torch.arange(s.T, device=DEV)
    seq = torch.searchsorted(s.cu_dev[1:].long().contiguous(), tok, right=True)
    return o[seq, tok - start[seq]].to(s.q.dtype)


# ------------------------------------------------------------------ prompt --

def _run_prompt(s):
    case = s.case
    if own:
        s.lib.attn_prompt_dev(s.type, case["dim"], s.hq, s.hk, s.hv, s.ho, s.cu_dev.data_ptr(), case["n_seq"], s.rows,
                              s.scale)
        return s.out
    T, H, kv, D = case["T"], case["heads"], case["kv"], case["dim"]
    G = H // kv
    q = s.q[:T].float().permute(1, 0, 2).reshape(kv, G * T, D)
    k, v = (t[:T].float().permute(1, 0, 2).contiguous() for t in (s.k, s.v))
    score = torch.matmul(q, k.transpose(1, 2).contiguous()).reshape(kv, G, T, T) * s.scale
    tok = torch.arange(T, device=DEV)
    seq = torch.searchsorted(s.cu_dev[1:].long().contiguous(), tok, right=True)
    seen = (tok[None] <= tok[:, None]) & (seq[None] == seq[:, None])
    score = score.masked_fill_(~seen, float("-inf"))
    p = torch.exp_(score.sub_(score.amax(-1, keepdim=True)))
    p = p.div_(p.sum(-1, keepdim=True)).reshape(kv, G * T, T)
    o = torch.matmul(p, v).reshape(H, T, D).permute(1, 0, 2)
    return torch.cat([o, o.new_zeros(case["pad"], H, D)]).to(s.q.dtype)


# -------------------------------------------------------------------- work --

def work(case):
    k = case["kind"]
    size = 4 if case.get("type") == "f32" else 2
    if k == "rope":
        n = case["T"] * (case["heads"] + case["kv"])
        return {"bytes": 2 * size * n * case["dim"] + 4 * case["T"] * len(case["axes"].split(",")), "flops": 3 * n * case["rot"]}
    if k == "slots":
        held, new, ended = _slot_lens(case)
        back = int(_ceil(held, case["block"])[ended].sum())
        take = int((_ceil(held + new, case["block"]) - _ceil(held, case["block"]))[~ended].sum())
        return {"bytes": 4 * (2 * case["T"] + 5 * case["n_seq"] + 2 * (back + take)), "flops": 4 * case["T"]}
    row = case["kv"] * 2 * (case["dim"] // 2 + case["dim"] // 16)       # a token's bytes in the cache
    if k == "append":
        n = 2 * case["T"] * case["kv"] * case["dim"]
        return {"bytes": size * n + 2 * case["T"] * row + 4 * n + 8 * case["T"], "flops": 8 * n}
    if k == "kv4":
        lens, ask = _kv_lens(case)
        seen = float(np.sum(ask * lens - ask * (ask - 1) // 2))
        return {"bytes": int(lens.sum()) * row + 2 * size * int(ask.sum()) * case["heads"] * case["dim"],
                "flops": 4 * seen * case["heads"] * case["dim"]}
    lens = _prompt_lens(case)
    return {"bytes": size * case["T"] * 2 * (case["heads"] + case["kv"]) * case["dim"],
            "flops": 4 * float(np.sum(lens * (lens + 1) // 2)) * case["heads"] * case["dim"]}


# ------------------------------------------------------------------- exact --

def _softmax64(score, live):
    """Weights [rows, keys] of float64 scores, live keys only."""
    score = torch.where(live, score, torch.full_like(score, -math.inf))
    e = torch.where(live, torch.exp(score - score.max(dim=1, keepdim=True).values), torch.zeros_like(score))
    return e / e.sum(1, keepdim=True)


def _exact_rope(s):
    case, out = s.case, []
    sizes = [int(a) for a in case["axes"].split(",")]
    left, axis, a = list(sizes), [], 0
    while sum(left):                    # pair by pair
        while not left[a]:
            a = (a + 1) % len(sizes)
        axis.append(a)
        left[a] -= 1
        a = (a + 1) % len(sizes) if case["turns"] else a
    i = np.arange(case["rot"] // 2)
    angle = s.pos.cpu().numpy().astype(np.float64)[axis].T * case["theta"] ** (-2.0 * i / case["rot"])
    ii, jj = (2 * i, 2 * i + 1) if case["adjacent"] else (i, i + case["rot"] // 2)
    for x in (s.q, s.k):
        x = x[..., :case["dim"]].double().cpu().numpy()
        y = x.copy()
        c, n = np.cos(angle)[:, None], np.sin(angle)[:, None]
        y[..., ii] = x[..., ii] * c - x[..., jj] * n
        y[..., jj] = x[..., ii] * n + x[..., jj] * c
        out.append(y)
    return tuple(out)


def _exact_slots(s):
    case, st = s.case, s.step
    bs, table, free, top = case["block"], st.table.copy(), st.free.copy(), st.n_free
    held = st.held.copy()
    for i in np.nonzero(st.ended)[0]:
        n = _ceil(int(held[i]), bs)
        free[top:top + n] = table[i, :n]
        top, held[i] = top + n, 0
    slot, pos, cu = np.full(case["T"], -1, np.int64), np.zeros(case["T"], np.int64), [0]
    for i in range(case["n_seq"]):
        for c in range(_ceil(int(held[i]), bs), _ceil(int(held[i] + st.new[i]), bs)):
            top -= 1
            table[i, c] = free[top]
        p = np.arange(held[i], held[i] + st.new[i])
        slot[cu[-1]:cu[-1] + len(p)] = table[i, p // bs].astype(np.int64) * bs + p % bs
        pos[cu[-1]:cu[-1] + len(p)] = p
        cu.append(cu[-1] + len(p))
    whole = lambda a: np.asarray(a, dtype=np.int32)  # noqa: E731
    return {"table": table, "free": free, "slot": whole(slot), "pos": whole(pos), "cu": whole(cu),
            "len": whole(held + st.new), "n_free": whole([top]), "status": np.zeros(2, np.int32)}


def _exact_append(s):
    out = []
    live = (s.slot >= 0).cpu().numpy()
    for x in (s.k, s.v):
        x = x.double().cpu().numpy().reshape(x.shape[0], x.shape[1], -1, GROUP)
        lo, hi = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
        d = ((hi - lo).astype(np.float32) / np.float32(15)).astype(np.float16).astype(np.float64)
        m = lo.astype(np.float16).astype(np.float64)
        code = np.clip(np.rint(((x - m).astype(np.float32) / d.astype(np.float32)).astype(np.float64)), 0, 15)
        out.append((d * code + m).reshape(s.k.shape) * live[:, None, None])
    return tuple(out)


def _exact_kv4(s):
    case = s.case
    H, kv, D, bs = case["heads"], case["kv"], case["dim"], case["block"]
    G, ng = H // kv, D // GROUP
    c = torch.arange(D, device=DEV)
    g, r = c // 64, c % 64
    k_byte = (r // 8 % 4) * (D // 8) + g * 8 + (r // 32) * 4 + (r % 8) // 2      # where a channel's code lies in a token's row
    v_byte = (r // 4) * (D // 32) + g * 2 + (r % 4) // 2
    half = bs * (D // 2 + D // 16)
    out = torch.empty((s.T, H, D), dtype=torch.float64, device=DEV)
    for i, (n, a) in enumerate(zip(s.lens.tolist(), s.ask.tolist())):
        if not a:
            continue
        t = torch.arange(n, device=DEV)
        page, off = s.table[i].long()[t // bs], t % bs
        seen = t[None] <= n - a + torch.arange(a, device=DEV)[:, None]
        for h in range(kv):
            piece = s.cache[:, h]
            vals = []
            for base, byte in ((0, k_byte), (half, v_byte)):
                b = piece[page[:, None], base + off[:, None] * (D // 2) + byte]
                code = torch.where(c % 2 == 1, b >> 4, b & 15).double()
                at = base + bs * D // 2 + (off[:, None] * ng + g) * 4
                d, m = (piece[page[:, None], at + o].to(torch.int32) | (piece[page[:, None], at + o + 1].to(torch.int32) << 8)
                        for o in (0, 2))
                d, m = (x.to(torch.int16).view(torch.float16).double() for x in (d, m))
                vals.append(code * d + m)
            for j in range(G):
                q = s.q[s.cu[i]:s.cu[i + 1], h * G + j].double()
                out[s.cu[i]:s.cu[i + 1], h * G + j] = _softmax64(q @ vals[0].T * s.scale, seen) @ vals[1]
    return out


def _exact_prompt(s):
    case = s.case
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=DEV)
    for a, b in zip(s.cu[:-1].tolist(), s.cu[1:].tolist()):
        if a == b:
            continue
        seen = torch.ones((b - a, b - a), dtype=torch.bool, device=DEV).tril()
        for h in range(case["heads"]):
            j = h * case["kv"] // case["heads"]
            w = _softmax64(s.q[a:b, h].double() @ s.k[a:b, j].double().T * s.scale, seen)
            out[a:b, h] = w @ s.v[a:b, j].double()
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    return {"rope": _exact_rope, "slots": _exact_slots, "append": _exact_append, "kv4": _exact_kv4,
            "prompt": _exact_prompt}[case["kind"]](s)
