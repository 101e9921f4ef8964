"""What the recurrent layers' entries and the log probabilities refuse before they touch a
device (CPU: a valid call gets as far as the missing device)."""
import ctypes as C

import pytest

ARG, NODEV = -2, -3
A = 1 << 32          # addresses that no check follows
FAR = 1 << 28


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


def conv_call(qm, **k):
    at = [A + i * FAR for i in range(9)]
    c = qm.Conv(k.get("channels", 96), k.get("width", 4), 1, k.get("n_slot", 5), k.get("weight", at[0]), k.get("bias", at[1]),
                k.get("state", at[2]))
    return qm.lib().qmag_conv_dev(None if k.get("none") else C.byref(c), k.get("type", 0), k.get("x", at[3]), k.get("xs", 96),
                                  k.get("out", at[4]), k.get("os", 96), k.get("slot", at[5]), k.get("len", at[6]),
                                  k.get("cu", at[7]), k.get("n_seq", 3), k.get("T", 10))


@pytest.mark.parametrize("bad", [
    dict(none=True), dict(type=12), dict(type=2), dict(channels=0), dict(channels=(1 << 20) + 1, xs=1 << 21, os=1 << 21),
    dict(width=1), dict(width=5), dict(n_slot=-1), dict(T=-1), dict(n_seq=-1), dict(n_seq=4097), dict(weight=None),
    dict(weight=A + 2), dict(bias=A + 1), dict(state=None), dict(state=A + 2), dict(slot=None), dict(slot=A + 1), dict(cu=None),
    dict(cu=A + 2), dict(len=A + 3), dict(x=None), dict(x=A + 3 * FAR + 2), dict(out=None), dict(xs=-1), dict(os=95),
    dict(xs=1 << 58), dict(out=A + 3 * FAR), dict(out=A + 3 * FAR + 4 * 96 * 9),      # over x
    dict(state=A + 3 * FAR), dict(state=A + 4 * FAR), dict(state=A + 5 * FAR), dict(state=A + 6 * FAR), dict(state=A + 7 * FAR),
    dict(state=A), dict(out=A), dict(out=A + FAR), dict(out=A + 5 * FAR), dict(out=A + 6 * FAR), dict(out=A + 7 * FAR + 12),
])
def test_conv_refusals(lib, bad):
    assert conv_call(lib, **bad) == ARG, lib.lib().qmag_last_error()


@pytest.mark.parametrize("good", [
    dict(), dict(type=1), dict(type=30), dict(width=2), dict(bias=None), dict(len=None), dict(T=0), dict(n_seq=0),
    dict(n_seq=0, cu=None, slot=None), dict(n_slot=0, state=None, slot=None), dict(xs=0), dict(xs=8192, os=100),
    dict(xs=192, os=192, out=A + 3 * FAR + 4 * 96),                                   # beside x in its rows
    dict(T=1, os=0), dict(T=2 ** 31 - 1),
])
def test_conv_accepted(lib, good):
    if good.get("T") == 2 ** 31 - 1:
        good = dict(good, out=A << 12, state=A << 13, weight=A << 14, bias=None, slot=A << 15, len=None, cu=(A << 15) + FAR)
    assert conv_call(lib, **good) == NODEV, lib.lib().qmag_last_error()


def linattn_call(qm, **k):
    at = [A + i * FAR for i in range(12)]
    dk, dv, H, K = k.get("dk", 128), k.get("dv", 64), k.get("heads", 6), k.get("keys", 3)
    a = qm.Linattn(H, dk, dv, k.get("delta", 1), k.get("turns", 0), k.get("eps", 1e-6), k.get("n_slot", 4), k.get("state", at[0]))
    views = [qm.heads(v) for v in (k.get("q", (at[1], K, 2000, 128)), k.get("k", (at[2], K, 2000, 128)),
                                   k.get("v", (at[3], H, 2000, 64)), k.get("out", (at[4], H, 2000, 64)))]
    if k.get("null") is not None:
        views[k["null"]] = None
    return qm.lib().qmag_linattn_dev(None if k.get("none") else C.byref(a), k.get("type", 0), *views, k.get("decay", at[5]),
                                     k.get("beta", at[6]), k.get("slot", at[7]), k.get("len", at[8]), k.get("cu", at[9]),
                                     k.get("n_seq", 3), k.get("T", 10), k.get("scale", 0.1))


@pytest.mark.parametrize("bad", [
    dict(none=True), dict(null=0), dict(null=1), dict(null=2), dict(null=3), dict(type=12), dict(type=-1), dict(dk=96), dict(dk=0),
    dict(dk=512), dict(dv=0), dict(dv=8), dict(dv=72), dict(dv=272), dict(heads=0), dict(heads=4097), dict(n_slot=-1),
    dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(scale=float("nan")), dict(scale=float("inf")),
    dict(T=-1), dict(n_seq=-1), dict(n_seq=4097), dict(state=None), dict(state=A + 8), dict(slot=None), dict(slot=A + 2),
    dict(cu=None), dict(cu=A + 1), dict(len=A + 2), dict(decay=A + 2), dict(beta=A + 1),
    dict(q=(None, 3, 2000, 128)), dict(q=(A + 2, 3, 2000, 128)), dict(q=(A + FAR, 2, 2000, 128)), dict(q=(A + FAR, 3, -1, 128)),
    dict(k=(A + 2 * FAR, 2, 2000, 128)), dict(q=(A + FAR, 4, 2000, 128), k=(A + 2 * FAR, 4, 2000, 128)),
    dict(q=(A + FAR, 0, 2000, 128), k=(A + 2 * FAR, 0, 2000, 128)), dict(v=(A + 3 * FAR, 3, 2000, 64)),
    dict(out=(A + 4 * FAR, 3, 2000, 64)), dict(out=(A + 4 * FAR, 6, 2000, 63)), dict(out=(A + 4 * FAR, 6, 100, 64)),
    dict(out=(A + FAR, 6, 2000, 64)), dict(out=(A + 2 * FAR + 4, 6, 2000, 64)), dict(out=(A + 3 * FAR, 6, 2000, 64)),
    dict(out=(A, 6, 2000, 64)), dict(out=(A + 5 * FAR, 6, 2000, 64)), dict(out=(A + 6 * FAR, 6, 2000, 64)),
    dict(out=(A + 7 * FAR, 6, 2000, 64)), dict(out=(A + 8 * FAR, 6, 2000, 64)), dict(out=(A + 9 * FAR, 6, 2000, 64)),
    dict(state=A + FAR), dict(state=A + 2 * FAR), dict(state=A + 3 * FAR), dict(state=A + 5 * FAR), dict(state=A + 6 * FAR),
    dict(state=A + 7 * FAR), dict(state=A + 8 * FAR), dict(state=A + 9 * FAR),
])
def test_linattn_refusals(lib, bad):
    assert linattn_call(lib, **bad) == ARG, lib.lib().qmag_last_error()


@pytest.mark.parametrize("good", [
    dict(), dict(type=1), dict(type=30), dict(dk=64), dict(dk=256, q=(A + FAR, 3, 2000, 256), k=(A + 2 * FAR, 3, 2000, 256)),
    dict(dv=16), dict(dv=48), dict(delta=0, beta=None), dict(decay=None), dict(len=None), dict(eps=0.0), dict(T=0), dict(n_seq=0),
    dict(n_seq=0, cu=None, slot=None), dict(n_slot=0, state=None, slot=None), dict(turns=1),
    # q, k, v and out side by side in one row
    dict(q=(A + FAR, 3, 2000, 128), k=(A + FAR + 4 * 384, 3, 2000, 128), v=(A + FAR + 4 * 768, 6, 2000, 64),
         out=(A + FAR + 4 * 1152, 6, 2000, 64)),
    # out where a key head's second half would be, heads apart by whole keys
    dict(keys=6, q=(A + FAR, 6, 1920, 192), k=(A + 2 * FAR, 6, 2000, 128), out=(A + FAR + 4 * 128, 6, 1920, 192)),
])
def test_linattn_accepted(lib, good):
    assert linattn_call(lib, **good) == NODEV, lib.lib().qmag_last_error()


def logprobs_call(qm, **k):
    at = [A + i * FAR for i in range(6)]
    return qm.lib().qmag_logprobs_dev(k.get("vocab", 1000), k.get("type", 0), k.get("x", at[0]), k.get("stride", 1000),
                                      k.get("token", at[1]), k.get("T", 7), k.get("top", 5), k.get("logprob", at[2]),
                                      k.get("entropy", at[3]), k.get("id", at[4]), k.get("val", at[5]))


@pytest.mark.parametrize("bad", [
    dict(type=12), dict(vocab=0), dict(T=-1), dict(top=-1), dict(top=65), dict(vocab=3, top=4), dict(x=None), dict(x=A + 2),
    dict(type=1, x=A + 1), dict(stride=-1), dict(stride=1 << 58), dict(token=None), dict(token=A + 1), dict(logprob=A + 2),
    dict(entropy=A + 2), dict(id=None), dict(val=None), dict(id=A + 1), dict(val=A + 3),
    dict(logprob=A), dict(entropy=A + 4000), dict(id=A + 27996), dict(val=A), dict(logprob=A + FAR), dict(entropy=A + FAR + 24),
    dict(id=A + FAR), dict(val=A + FAR), dict(entropy=A + 2 * FAR), dict(id=A + 3 * FAR + 24), dict(val=A + 4 * FAR + 136),
])
def test_logprobs_refusals(lib, bad):
    assert logprobs_call(lib, **bad) == ARG, lib.lib().qmag_last_error()


@pytest.mark.parametrize("good", [
    dict(), dict(type=1), dict(type=30), dict(T=0), dict(top=0, id=None, val=None), dict(logprob=None, token=None),
    dict(entropy=None), dict(logprob=None, entropy=None, token=None, top=0), dict(top=64), dict(vocab=1, top=1), dict(stride=0),
    dict(stride=1100, entropy=A + 4000), dict(vocab=2 ** 31 - 1, stride=2 ** 31 - 1, T=1, logprob=A << 4, entropy=A << 5,
                                              id=A << 6, val=A << 7, token=A << 8),
])
def test_logprobs_accepted(lib, good):
    assert logprobs_call(lib, **good) == NODEV, lib.lib().qmag_last_error()
