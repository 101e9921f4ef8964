"""What the attention entries refuse before they touch a device (CPU: a valid
call gets as far as the missing device)."""
import ctypes as C

import pytest

ARG, NODEV = -2, -3


@pytest.fixture(scope="module")
def lib():
    import os

    import qmag
    if not os.path.exists(qmag.LIB_PATH):
        import build as b
        b.build()
    L = qmag.lib()
    if L.qmag_init(0) == 0:
        pytest.skip("a gfx950 GPU is visible")
    return qmag


A = 1 << 20          # addresses that no check follows


def rope_call(qm, **k):
    D = k.pop("dim", 128)
    r = qm.Rope.make(D, k.pop("rot", 64), k.pop("sections", (16, 16)), theta=k.pop("theta", 1e4))
    for name in ("n_axes", "n_rot"):
        if name in k:
            setattr(r, name, k.pop(name))
    src = k.pop("src", ((A, 4, 512, 128), (A + (1 << 20), 2, 256, 128)))
    dst = k.pop("dst", src)
    s, d = qm.heads(*src), qm.heads(*dst)
    return qm.lib().qmag_rope_dev(C.byref(r), k.get("pos", A), k.get("T", 5), k.get("type", 0), s, d, k.get("views", len(src)))


@pytest.mark.parametrize("bad", [
    dict(pos=None), dict(pos=A + 1), dict(T=-1), dict(type=2), dict(type=12), dict(views=0), dict(views=3), dict(dim=1),
    dict(dim=2048), dict(rot=63, sections=(16, 15)), dict(rot=0, sections=(0,)), dict(rot=256, sections=(128,)),
    dict(sections=(16, 15)), dict(sections=(-1, 33)), dict(n_axes=0), dict(n_axes=5), dict(theta=0.0), dict(theta=-1.0),
    dict(theta=float("nan")), dict(theta=float("inf")),
    dict(src=((None, 4, 512, 128),)), dict(src=((A + 2, 4, 512, 128),)), dict(src=((A, -1, 512, 128),)),
    dict(src=((A, 5000, 512, 128),)), dict(src=((A, 4, -512, 128),)),
    dict(src=((A, 4, 1 << 40, 128),), T=2 ** 31 - 1), dict(src=((A, 4, 128, 1 << 57),)),   # places beyond 64 bits
    dict(src=((A, 4, 512, 64),)),                                             # heads on one another, written
    dict(src=((A, 4, 500, 128),)),                                            # tokens on one another
    dict(src=((A, 4, 512, 128),), dst=((A + 4, 4, 512, 128),)),               # over its source, shifted
    dict(src=((A, 4, 512, 128),), dst=((A + 65536, 2, 512, 128),)),           # fewer heads
    dict(src=((A, 4, 512, 128), (A + 1024, 2, 512, 128))),                    # k within q
])
def test_rope_refusals(lib, bad):
    assert rope_call(lib, **bad) == ARG, lib.lib().qmag_last_error()


@pytest.mark.parametrize("good", [
    dict(), dict(T=0), dict(type=1), dict(type=30), dict(T=0, pos=None),
    dict(src=((A, 4, 1536, 256), (A + 4096, 2, 1536, 128))),                  # q beside a gate, then k, in one row
    dict(src=((A, 4, 1024, 256),), dst=((A + 512, 4, 1024, 256),)),           # into the other half of every head
    dict(src=((A, 4, 128, 640),)),                                            # whole heads one behind another
])
def test_rope_accepted(lib, good):
    assert rope_call(lib, **good) == NODEV, lib.lib().qmag_last_error()


def kv4(qm, **k):
    return qm.Kv4(k.get("data", A), k.get("n_block", 64), k.get("block_size", 16), k.get("n_kv", 2), k.get("head_dim", 128))


CACHE_BAD = [dict(data=None), dict(data=A + 8), dict(n_block=0), dict(n_block=1 << 28), dict(block_size=8), dict(block_size=48),
             dict(block_size=512), dict(n_kv=0), dict(n_kv=5000), dict(head_dim=96), dict(head_dim=0), dict(head_dim=512)]


@pytest.mark.parametrize("bad", CACHE_BAD)
def test_cache_refusals(lib, bad):
    L, c = lib.lib(), kv4(lib, **bad)
    h = lib.heads((A, 2, 256, 128))
    assert L.qmag_kv4_append_dev(C.byref(c), 0, h, h, A, 4) == ARG
    assert L.qmag_kv4_read_dev(C.byref(c), A, 4, A, A) == ARG
    t = lib.KvTable(1, 4, c.block_size, c.n_block, A, A)
    q, o = lib.heads((A, 2, 256, 128)), lib.heads((A << 4, 2, 256, 128))
    assert L.qmag_attn_kv4_dev(C.byref(c), C.byref(t), 0, q, o, A, A, 4, 1.0) == ARG
    n = C.c_size_t()
    if "data" not in bad and "n_block" not in bad:
        assert L.qmag_kv4_block_bytes(C.byref(c), C.byref(n)) == ARG


def test_block_bytes(lib):
    for D in (64, 128, 256):
        c = lib.Kv4(None, 0, 32, 3, D)
        assert lib.kv4_block_bytes(c) == 3 * 32 * 2 * (D // 2 + D // 16)


@pytest.mark.parametrize("k,v,slot,T,typ", [
    ((A, 3, 384, 128), (A, 2, 256, 128), A, 4, 0), ((A, 2, 256, 128), (A, 1, 128, 128), A, 4, 0),
    ((A, 2, 256, 128), (None, 2, 256, 128), A, 4, 0), ((A, 2, 256, 128), (A, 2, 256, 128), None, 4, 0),
    ((A, 2, 256, 128), (A, 2, 256, 128), A + 2, 4, 0), ((A, 2, 256, 128), (A, 2, 256, 128), A, -1, 0),
    ((A, 2, 256, 128), (A, 2, 256, 128), A, 4, 3), ((A + 1, 2, 256, 128), (A, 2, 256, 128), A, 4, 1),
])
def test_append_refusals(lib, k, v, slot, T, typ):
    c = kv4(lib)
    assert lib.lib().qmag_kv4_append_dev(C.byref(c), typ, lib.heads(k), lib.heads(v), slot, T) == ARG
    ok = lib.heads((A, 2, 256, 128))
    assert lib.lib().qmag_kv4_append_dev(C.byref(c), 1, ok, ok, A, 4) == NODEV


def table(qm, **k):
    return qm.KvTable(k.get("n_seq", 3), k.get("max_blocks", 4), k.get("block_size", 16), k.get("n_block", 64),
                      k.get("table", A), k.get("free_list", A))


@pytest.mark.parametrize("bad", [dict(n_seq=-1), dict(n_seq=4097), dict(max_blocks=0), dict(block_size=24), dict(n_block=0),
                                 dict(n_block=1 << 27, block_size=32), dict(table=None), dict(free_list=None)])
def test_bookkeeping_refusals(lib, bad):
    L, t = lib.lib(), table(lib, **bad)
    p = [A + 4096 * i for i in range(10)]
    assert L.qmag_kv_release_dev(C.byref(t), *p[:6]) == ARG
    assert L.qmag_kv_assign_dev(C.byref(t), p[0], p[1], p[2], 5, *p[3:9]) == ARG


def test_bookkeeping_pointers(lib):
    L, t = lib.lib(), table(lib)
    p = [A + 4096 * i for i in range(10)]
    assert L.qmag_kv_release_dev(C.byref(t), *p[:6]) == NODEV
    assert L.qmag_kv_assign_dev(C.byref(t), p[0], p[1], p[2], 5, *p[3:9]) == NODEV
    for i in range(6):
        assert L.qmag_kv_release_dev(C.byref(t), *[None if j == i else x for j, x in enumerate(p[:6])]) == ARG
    assert L.qmag_kv_release_dev(C.byref(t), p[0], p[1], p[2], p[0], p[4], p[5]) == ARG     # lengths over themselves
    assert L.qmag_kv_release_dev(C.byref(t), p[0], p[1], p[2], p[3], p[2], p[5]) == ARG
    assert L.qmag_kv_assign_dev(C.byref(t), p[0], p[1], p[2], -1, *p[3:9]) == ARG
    assert L.qmag_kv_assign_dev(C.byref(t), p[0], p[1], p[2], 5, p[3], p[4], p[5], p[0], p[7], p[8]) == ARG
    assert L.qmag_kv_assign_dev(C.byref(t), p[0], p[1], p[2], 5, p[3], p[4], p[5], p[6], p[2], p[8]) == ARG
    assert L.qmag_kv_assign_dev(C.byref(t), p[0], p[1], p[2], 5, None, *p[4:9]) == ARG
    assert L.qmag_kv_assign_dev(C.byref(t), p[0], p[1], p[2], 0, None, None, *p[5:9]) == NODEV


def test_bookkeeping_results_over_inputs(lib):
    """What is written meets neither an input nor another result, by a part of it either."""
    L, t = lib.lib(), table(lib, n_seq=10)
    p = [A + 4096 * i for i in range(10)]
    ok = dict(zip(("len", "ended", "n_free", "len_next", "n_free_next", "status"), p))
    rel = lambda **k: L.qmag_kv_release_dev(C.byref(t), *dict(ok, **k).values())  # noqa: E731
    assert rel() == NODEV and rel(ended=p[0]) == NODEV and rel(len_next=p[0] + 40) == NODEV
    for k in (dict(len_next=p[0] + 36), dict(len_next=p[1]), dict(status=p[0] + 4), dict(status=p[2]), dict(status=p[4]),
              dict(n_free_next=p[3] + 36), dict(len=p[0] + 2), dict(status=p[5] + 1)):
        assert rel(**k) == ARG, k
    ok = dict(zip(("len", "new", "n_free"), p), T=20, slot=p[3], pos=p[4], cu=p[5], len_next=p[6], n_free_next=p[7], status=p[8])
    assign = lambda **k: L.qmag_kv_assign_dev(C.byref(t), *dict(ok, **k).values())  # noqa: E731
    assert assign() == NODEV and assign(pos=p[3] + 80) == NODEV and assign(len_next=p[5] + 44) == NODEV
    for k in (dict(pos=p[3]), dict(pos=p[3] + 76), dict(len_next=p[5] + 40), dict(cu=p[1]), dict(len_next=p[1] - 36),
              dict(status=p[2]), dict(n_free_next=p[8]), dict(slot=p[0] + 4), dict(cu=p[5] + 2)):
        assert assign(**k) == ARG, k


@pytest.mark.parametrize("bad", [dict(T=-1), dict(T=(1 << 22) + 1), dict(n_seq=5000), dict(cu=None), dict(cu=A + 1), dict(len=None),
                                 dict(len=A + 2), dict(table=None), dict(max_blocks=0), dict(max_blocks=1 << 27), dict(n_block=63),
                                 dict(tbs=32), dict(q=(A, 3, 384, 128)), dict(out=(A << 4, 8, 1024, 128)), dict(q=(A, 0, 0, 0)),
                                 dict(out=(A + 64, 4, 512, 128)), dict(out=(A << 4, 4, 512, 0)), dict(type=5)])
def test_attn_kv4_refusals(lib, bad):
    def call(**k):
        c = kv4(lib)
        t = lib.KvTable(k.get("n_seq", 3), k.get("max_blocks", 4), k.get("tbs", 16), k.get("n_block", 64), k.get("table", A), None)
        q, o = lib.heads(k.get("q", (A, 4, 512, 128))), lib.heads(k.get("out", (A << 4, 4, 512, 128)))
        return lib.lib().qmag_attn_kv4_dev(C.byref(c), C.byref(t), k.get("type", 0), q, o, k.get("cu", A), k.get("len", A),
                                           k.get("T", 5), 1.0)
    assert call() == NODEV and call(T=0, cu=None, len=None) == NODEV
    assert call(**bad) == ARG, lib.lib().qmag_last_error()


@pytest.mark.parametrize("bad", [dict(type=8), dict(dim=96), dict(dim=512), dict(T=-1), dict(T=(1 << 22) + 1), dict(n_seq=-1),
                                 dict(n_seq=4097), dict(cu=None), dict(cu=A + 2), dict(k=(A << 1, 3, 384, 128)),
                                 dict(v=(A << 2, 1, 128, 128)), dict(out=(A, 4, 512, 128)), dict(out=(A << 1, 4, 512, 128)),
                                 dict(out=(A << 3, 4, 512, 100)), dict(k=(None, 2, 256, 128)), dict(k=(A << 1, 0, 0, 0))])
def test_attn_prompt_refusals(lib, bad):
    def call(**k):
        h = [lib.heads(k.get(n, (A << i, heads, heads * 128, 128))) for i, (n, heads) in
             enumerate((("q", 4), ("k", 2), ("v", 2), ("out", 4)))]
        return lib.lib().qmag_attn_prompt_dev(k.get("type", 0), k.get("dim", 128), *h, k.get("cu", A), k.get("n_seq", 2),
                                              k.get("T", 5), 1.0)
    assert call() == NODEV and call(T=0, cu=None) == NODEV and call(type=30) == NODEV
    assert call(**bad) == ARG, lib.lib().qmag_last_error()


def test_bookkeeping_results_over_the_lists(lib):
    """The table and the free list, which the workgroups of a call read and write, meet neither one
    another nor a result; the one that is written meets no input."""
    L = lib.lib()
    p = [A + 4096 * i for i in range(10)]
    T, F = A + (1 << 16), A + (1 << 17)                     # 10 x 4 and 64 words

    def rel(table=T, free=F, **k):
        t = lib.KvTable(10, 4, 16, 64, table, free)
        ok = dict(zip(("len", "ended", "n_free", "len_next", "n_free_next", "status"), p))
        return L.qmag_kv_release_dev(C.byref(t), *dict(ok, **k).values())

    def assign(table=T, free=F, **k):
        t = lib.KvTable(10, 4, 16, 64, table, free)
        ok = dict(zip(("len", "new", "n_free"), p), T=20, slot=p[3], pos=p[4], cu=p[5], len_next=p[6], n_free_next=p[7], status=p[8])
        return L.qmag_kv_assign_dev(C.byref(t), *dict(ok, **k).values())

    assert rel() == NODEV and assign() == NODEV
    assert rel(table=F - 160) == NODEV and rel(table=F - 156) == ARG and assign(free=T - 252) == ARG and assign(free=T - 256) == NODEV
    assert rel(table=T + 2) == ARG and assign(free=F + 1) == ARG
    for name in ("len_next", "n_free_next", "status"):
        assert rel(**{name: T + 156}) == ARG and rel(**{name: F + 252}) == ARG and rel(**{name: F + 256}) == NODEV, name
    for name in ("len", "ended", "n_free"):                 # the free list is written, the table is not
        assert rel(**{name: F + 4}) == ARG and rel(**{name: T}) == NODEV, name
    for name in ("slot", "pos", "cu", "len_next", "n_free_next", "status"):
        assert assign(**{name: T + 156}) == ARG and assign(**{name: F}) == ARG and assign(**{name: T + 160}) == NODEV, name
    for name in ("len", "new", "n_free"):                   # the table is written
        assert assign(**{name: T}) == ARG and assign(**{name: F}) == NODEV, name
    assert assign(T=0, slot=T, pos=F) == NODEV              # nothing of them is written


def test_attention_output_over_what_it_reads(lib):
    """The output meets neither lengths, table nor cache; beside them, between its own heads or tokens, it may lie."""
    L, out = lib.lib(), A << 4
    size = 64 * 16 * 2 * 2 * (64 + 8)

    def kv4_call(layout=(out, 4, 640, 160), **k):           # heads of 128 values of 4 bytes, 32 values between them
        c = kv4(lib, data=k.get("data", A))
        t = lib.KvTable(3, 4, 16, 64, k.get("table", A), None)
        q, o = lib.heads((A, 4, 512, 128)), lib.heads(layout)
        return L.qmag_attn_kv4_dev(C.byref(c), C.byref(t), 0, q, o, k.get("cu", A), k.get("len", A), 5, 1.0)

    assert kv4_call() == NODEV
    end = out + 4 * (4 * 640 + 3 * 160 + 128)
    for name, n in (("cu", 16), ("len", 12), ("table", 48)):
        for at in (out, out + 4 * 640, end - 4, out - n + 4, out + 4 * 100, out + 4 * (640 + 128) - 4):
            assert kv4_call(**{name: at}) == ARG, (name, at - out)
        for at in (out - n, end, out + 4 * 128, out + 4 * (2 * 640 + 160 + 128)):
            assert kv4_call(**{name: at}) == NODEV, (name, at - out)
        # heads one behind another: a token's values lie among them
        heads_major = (out, 4, 160, 1000)
        assert kv4_call(heads_major, **{name: out + 4 * (2 * 1000 + 160)}) == ARG
        assert kv4_call(heads_major, **{name: out + 4 * (1000 + 3 * 160 + 128)}) == NODEV
    assert kv4_call(data=out + 16) == ARG and kv4_call(data=out - size + 16) == ARG and kv4_call(data=out - size) == NODEV

    def prompt(cu):
        h = [lib.heads((a, n, n * 128, 128)) for a, n in ((A, 4), (A << 1, 2), (A << 2, 2), (A << 3, 4))]
        return L.qmag_attn_prompt_dev(0, 128, *h, cu, 2, 5, 1.0)
    assert prompt(A << 3) == ARG and prompt((A << 3) + 4 * 5 * 512 - 4) == ARG and prompt((A << 3) - 8) == ARG
    assert prompt((A << 3) + 4 * 5 * 512) == NODEV and prompt((A << 3) - 12) == NODEV


def test_read_results_over_what_it_reads(lib):
    L, c = lib.lib(), kv4(lib)
    k, v, s, n = A << 2, A << 3, A << 4, 4 * 2 * 128 * 4    # four tokens of two heads
    size = 64 * 16 * 2 * 2 * (64 + 8)
    read = lambda slot, k, v: L.qmag_kv4_read_dev(C.byref(c), slot, 4, k, v)  # noqa: E731
    assert read(s, k, v) == NODEV and read(s, k, k + n) == NODEV and read(s, k, k + n - 4) == ARG and read(s, k, k) == ARG
    assert read(k + n - 4, k, v) == ARG and read(v - 12, k, v) == ARG and read(k + n, k, v) == NODEV
    assert read(s, A, v) == ARG and read(s, k, A + size - 16) == ARG and read(s, k, A + size) == NODEV


@pytest.mark.parametrize("theta,ok", [(1e-320, False), (1e-306, False), (1e-300, True), (1e-3, True), (1.0, True), (1e300, True)])
def test_rope_frequencies_are_numbers(lib, theta, ok):
    """theta^(-2 i / n_rot) times the largest position has to stay in range: 0 times an infinity is no angle.
    (1e-300: 10^(300 x 126 / 128) 2^31 / 2 pi = 10^304.)"""
    assert rope_call(lib, theta=theta, rot=128, sections=(64,)) == (NODEV if ok else ARG)


def test_views_side_by_side_within_heads(lib):
    """[head][q's tokens, k's tokens, ...] in one buffer: apart, unless a token reaches into the next view."""
    S, D, T = 4096, 64, 8                                    # values to a head, of a token, tokens
    at = lambda i, n=2: (A + int(4 * i * T * D), n, D, S)    # noqa: E731
    assert rope_call(lib, dim=D, T=T, src=(at(0), at(1)), dst=(at(2), at(3))) == NODEV
    assert rope_call(lib, dim=D, T=T, src=(at(0), at(1)), dst=(at(2), at(2.5))) == ARG
    assert rope_call(lib, dim=D, T=T, src=(at(0), at(1)), dst=(at(0.5), at(3))) == ARG
    assert rope_call(lib, dim=D, T=T + 1, src=(at(0), at(1)), dst=(at(2), at(3))) == ARG
    assert rope_call(lib, dim=D, T=T, src=(at(0, 5), at(1, 1)), dst=(at(2, 5), at(3, 1))) == NODEV
    assert rope_call(lib, dim=D, T=T, src=(at(0, 5), at(1)), dst=(at(7, 5), at(8))) == ARG      # behind its head: in the next one's first view
