"""Refusals of the operators for several continuations of one prompt, without a GPU: every bad
argument is K2T_E_ARG before anything touches a device (where there is none, a call that passes its
checks ends in K2T_E_HIP)."""
import ctypes as C

import pytest

import branch_ref as R
import k2t

CTX = (C.c_char * 4096)()  # stands for a context: the checks come before its first use
P = 1 << 20  # an aligned address; nothing is read from it
ARG, HIP = -1, -2


def rows(kq=P, ks=P, vq=P, vs=P, cap=8, length=8):
    return k2t.KVRows(kq, ks, vq, vs, cap=cap, len=length)


def call(name, *args):
    a = [C.addressof(x) if isinstance(x, (k2t.KVRows, C.Array)) else x for x in args]
    return getattr(k2t.lib(), name)(*a)


def refused(name, good, bad):
    """Each {index: value} change of a good call is refused; returns the messages."""
    for change in bad:
        args = list(good)
        for i, v in change.items():
            args[i] = v
        assert call(name, *args) == ARG, (name, change)
        assert k2t.lib().k2t_last_error().decode()


BAD_CACHE = [rows(kq=0), rows(vs=0), rows(kq=P + 8), rows(vq=P + 1), rows(ks=P + 2), rows(vs=P + 1), rows(cap=0, length=0),
             rows(length=9), rows(length=-1), rows(cap=(1 << 24) + 1)]


def test_append_and_load():
    good = [CTX, 8, P, P, 256, 2, 3, 2, 128, P, None, rows()]
    refused("k2t_kv_append", good, [{0: None}, {1: 5}, {1: 16}, {2: None}, {3: None}, {2: P + 4}, {4: 255}, {4: 258}, {5: -1},
                                    {6: -1}, {7: 0}, {8: 96}, {9: None}, {11: None}, {5: 1 << 20, 6: 1 << 10},
                                    {6: 1 << 30, 7: 1 << 30, 4: 1 << 40}, {7: 1025, 4: 1 << 20}] +
            [{11: c} for c in BAD_CACHE])
    good = [CTX, 4, rows(), 2, 3, 2, 128, P, None, P, P, 256]
    refused("k2t_kv_load", good, [{0: None}, {1: 3}, {2: None}, {2: rows(ks=P + 2)}, {6: 32}, {7: None}, {9: None},
                                  {10: P + 8}, {11: 128}])
    if k2t.lib().k2t_device_count() == 0:
        assert call("k2t_kv_load", *good) == HIP
        assert call("k2t_kv_append", CTX, 8, None, None, 256, 0, 3, 2, 128, None, None, rows()) == 0  # nothing to do


def test_reorder():
    good = [CTX, 8, rows(), P, 2, 1, 4, 2, 64]
    refused("k2t_kv_reorder", good, [{0: None}, {1: 7}, {2: None}, {3: None}, {4: -1}, {5: -1}, {6: 0}, {6: 65}, {7: 0}, {8: 63},
                                     {4: 1 << 20, 5: 100}, {4: 1 << 30, 5: 1 << 30, 7: 16}, {7: 1 << 30},
                                     {2: rows(cap=1 << 24, length=1 << 24)}] +
            [{2: c} for c in BAD_CACHE])
    if k2t.lib().k2t_device_count() == 0:
        assert call("k2t_kv_reorder", *good) == HIP
        assert call("k2t_kv_reorder", CTX, 8, rows(length=0), P, 2, 1, 4, 2, 64) == 0


def test_attention():
    n = C.c_size_t()
    assert call("k2t_attn_shared_workspace", CTX, 1, 4, 8, 2, 64, 8, 8, C.byref(n)) == 0 and n.value >= 16
    good = [CTX, 8, P, 512, 1, 4, 8, 2, 64, rows(), rows(), 0.125, P, P, n.value]
    refused("k2t_attn_shared", good, [{0: None}, {1: 0}, {2: None}, {2: P + 4}, {3: 511}, {3: 514}, {3: 1 << 31}, {4: -1}, {5: 0}, {6: 7},
                                      {6: 2048}, {7: 0}, {8: 80}, {9: None, 10: None}, {12: None}, {12: P + 4}, {13: None},
                                      {13: P + 8}, {14: n.value - 1}, {4: 70000}, {11: -0.125}, {11: float("nan")}, {11: float("inf")},
                                      {4: 16000, 6: 1024}] +
            [{i: c} for c in BAD_CACHE for i in (9, 10)])
    refused("k2t_attn_shared_workspace", [CTX, 1, 4, 8, 2, 64, 8, 8, C.byref(n)],
            [{0: None}, {1: -1}, {2: 0}, {3: 9}, {5: 256}, {6: -1}, {7: -1}, {8: None}])
    if k2t.lib().k2t_device_count() == 0:
        assert call("k2t_attn_shared", *good) == HIP


@pytest.mark.parametrize("shape", [(1, 8, 32, 32, 64), (3, 8, 32, 8, 128), (1, 8, 32, 8, 128), (1, 8, 32, 4, 128),
                                   (1, 64, 32, 4, 128), (1, 1, 1, 1, 64), (1, 4, 9, 3, 64), (4, 64, 32, 8, 128), (2, 3, 40, 2, 64)])
def test_attention_workspace_serves_shorter_caches(shape):
    """k2t_attn_shared_workspace of the longest caches is enough for a call with any shorter ones (a longer
    cache may be cut into fewer parts than a shorter one), and no less than that of the shorter ones."""
    ctx = (C.c_int32 * 1024)(*[256] * 1024)  # a context of 256 CUs, on a device that no machine has

    def workspace(p, t):
        n = C.c_size_t()
        assert call("k2t_attn_shared_workspace", ctx, *shape, p, t, C.byref(n)) == 0
        return n.value

    def accepted(p, t, ws):
        n_seq, beams, nq, nkv, hd = shape
        pre, tail = (rows(cap=1 << 24, length=n) if n else None for n in (p, t))
        if not (p or t):
            pre = rows(length=0)
        rc = call("k2t_attn_shared", ctx, 8, P, nq * hd, *shape, pre, tail, 0.125, P, P, ws)
        assert rc in (ARG, HIP)
        return rc == HIP  # (past the checks: the device is the one that does not exist)

    lengths = [0, 1, 31, 45, 90, 127, 128, 129, 384, 385, 511, 700, 768, 769, 1000, 1153, 1280, 1400, 2048, 2100, 3840, 4100, 9000,
               65537, 1 << 20]
    for p, t in [(2100, 64), (2048, 64), (1400, 90), (45, 769), (1000, 385), (4100, 90), (0, 4100), (9000, 0), (1 << 20, 1 << 20),
                 (65537, 700)]:
        ws = workspace(p, t)
        for a in [n for n in lengths if n <= p]:
            for b in [n for n in lengths if n <= t]:
                assert accepted(a, b, ws), (p, t, a, b)
                assert workspace(a, b) <= ws, (p, t, a, b)


def test_select():
    n = C.c_size_t()
    assert call("k2t_beam_select_workspace", CTX, 2, 4, 1000, 8, C.byref(n)) == 0 and n.value >= 16
    good = [CTX, P, 1000, 1000, P, P, 2, 4, 8, 5, 2 * P, P, P, 2 * P, P, n.value]
    refused("k2t_beam_select", good, [{0: None}, {1: None}, {2: 0}, {2: 262145, 3: 262145}, {3: 999}, {4: None}, {6: -1}, {7: 0}, {7: 65}, {8: 0},
                                      {8: 129}, {9: -2}, {9: 1000}, {9: -1}, {10: None}, {11: None}, {12: None}, {14: None},
                                      {14: P + 8}, {15: n.value - 1}, {6: 20000}, {10: P + 64, 4: P + 64}, {13: P + 64, 5: P + 64}])
    refused("k2t_beam_select_workspace", [CTX, 2, 4, 1000, 8, C.byref(n)], [{0: None}, {2: 65}, {3: 0}, {4: 0}, {5: None}])
    if k2t.lib().k2t_device_count() == 0:
        assert call("k2t_beam_select", *good) == HIP


def test_the_reference_itself():
    """branch_ref on a case small enough to work out by hand."""
    import numpy as np
    x = np.array([[0.0, np.log(3.0)], [0.0, 0.0]], np.float32)
    s, t, p, d, _ = R.select(x, np.array([0.0, -0.1], np.float32), None, 1, 2, 3, -1)
    assert t.tolist() == [[1, 0, 1]] and p.tolist() == [[0, 1, 1]] and d.tolist() == [[0, 0, 0]]
    assert np.allclose(s, [[np.log(0.75), np.log(0.5) - 0.1, np.log(0.5) - 0.1]], atol=1e-6)
    # the inverse rotation undoes the oracle's, and a head's codes stand for the head
    import oracle as O
    rng = np.random.default_rng(0)
    head = rng.standard_normal(128).astype(np.float32)
    assert np.abs(R.unrotate(O.fwht64(head).astype(np.float64)) - head).max() < 1e-6
    for bits, step in ((8, 0.51 / 127), (4, 0.15)):  # (half a code step; half the NF4 codebook's widest gap)
        q, s = R.store(bits, head)
        off = R.values(bits, q[None], np.asarray(s)[None])[0] - O.fwht64(head)
        assert np.abs(off).max() <= step * np.abs(O.fwht64(head)).max()
