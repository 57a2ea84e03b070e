"""The operators for blocks of tokens without a GPU: rope plans, and refusals (every bad argument is
K2T_E_ARG before anything touches a device; where there is none, a call that passes its checks ends in K2T_E_HIP)."""
import ctypes as C

import numpy as np
import pytest

import block_ref as R
import k2t
from test_branch_args import BAD_CACHE, CTX, HIP, P, call, refused, rows

KINDS = {"plain": k2t.ROPE_PLAIN, "linear": k2t.ROPE_LINEAR, "base": k2t.ROPE_BASE, "ramp": k2t.ROPE_RAMP,
         "wave": k2t.ROPE_WAVE}


def no_gpu():
    return k2t.lib().k2t_device_count() == 0


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("rot,theta", [(64, 100000.0), (128, 1e6), (90, 10000.0), (4, 130000.0), (2, 500.0)])
def test_plan_holds_the_formulas_frequencies(kind, rot, theta):
    if kind == "base" and rot == 2:
        return
    for factor, original, low, high in ((16.0, 8192, 0.0, 0.0), (3.5, 1000, 0.5, 20.0), (0.5, 4096, 1.0, 4.0)):
        p = k2t.RopePlan(k2t.ROPE_HALF, rot, theta, KINDS[kind], factor, original, low, high)
        want, scale = R.turns(rot, theta, kind, factor, original, low, high)
        got = np.array(p.turns[:rot // 2])
        # pow, a quotient, a blend and another quotient: a few roundings of 2^-53; pow's exponent -2 i / d is rounded
        # too, which the logarithm of theta multiplies (ln 1e6 = 14)
        assert (np.abs(got - want) <= 2.0 ** -53 * (40 + 8) * want).all()
        assert abs(p.scale - scale) <= 2.0 ** -50 and p.layout == k2t.ROPE_HALF and p.rot_dim == rot


def test_plan_refusals():
    good = dict(layout=0, rot_dim=64, scaling=k2t.ROPE_RAMP, original=4096, theta=1e5, factor=4.0, low=1.0, high=32.0)
    nan, inf = float("nan"), float("inf")

    def rc(**change):
        cfg, out = k2t.RopeConfig(**dict(good, **change)), k2t.RopePlan.__new__(k2t.RopePlan)
        return k2t.lib().k2t_rope_plan_make(C.addressof(cfg), C.addressof(out))

    assert rc() == 0
    for bad in (dict(layout=2), dict(layout=-1), dict(rot_dim=0), dict(rot_dim=63), dict(rot_dim=130), dict(scaling=5),
                dict(scaling=-1), dict(theta=1.0), dict(theta=0.5), dict(theta=nan), dict(theta=inf), dict(factor=0.0),
                dict(factor=-1.0), dict(factor=nan), dict(factor=inf), dict(original=0), dict(low=-1.0), dict(low=2.0, high=2.0),
                dict(low=nan), dict(high=inf), dict(scaling=k2t.ROPE_BASE, rot_dim=2), dict(scaling=k2t.ROPE_LINEAR, factor=0.01)):
        assert rc(**bad) == -1, bad
    assert rc(scaling=k2t.ROPE_PLAIN, factor=nan, original=0, low=nan) == 0  # (not looked at)
    assert call("k2t_rope_plan_make", None, None) == -1


def plan(rot=64, **change):
    p = k2t.RopePlan(k2t.ROPE_HALF, rot, 1e4)
    for n, v in change.items():
        if n == "turns":
            p.turns[3] = v
        else:
            setattr(p, n, v)
    return p


def test_rope():
    def at(p):
        keep.append(p)
        return C.addressof(p)
    keep = []
    good = [CTX, P, 256, 2, 3, 4, 64, P, None, None, at(plan()), P, 256]
    refused("k2t_rope", good, [{0: None}, {1: None}, {1: P + 4}, {2: 255}, {2: 258}, {3: -1}, {3: 65536}, {4: -1}, {5: 0},
                               {5: 2049, 2: 1 << 20, 12: 1 << 20}, {6: 96}, {6: 32}, {7: None}, {10: None}, {11: None}, {11: P + 8},
                               {12: 128}, {12: 260}, {12: 258}, {3: 60000, 4: 60000}, {2: 1 << 40, 12: 1 << 40},
                               {10: at(plan(128))}, {10: at(plan(layout=2))}, {10: at(plan(rot_dim=0))}, {10: at(plan(rot_dim=7))},
                               {10: at(plan(scale=float("nan")))}, {10: at(plan(turns=1.5))}, {10: at(plan(turns=float("nan")))}])
    if no_gpu():
        assert call("k2t_rope", *good) == HIP
        for nothing in ({3: 0}, {4: 0}):
            args = list(good)
            args[1] = args[7] = args[11] = None
            for i, v in nothing.items():
                args[i] = v
            assert call("k2t_rope", *args) == 0


def test_attention():
    n = C.c_size_t()
    shape = [2, 5, 8, 2, 64]
    assert call("k2t_attn_tokens_workspace", CTX, *shape, 8, C.byref(n)) == 0 and n.value >= 16
    good = [CTX, 8, P, 512, *shape, P, None, None, rows(), 0.125, P, P, n.value]
    refused("k2t_attn_tokens", good, [{0: None}, {1: 5}, {2: None}, {2: P + 4}, {3: 511}, {3: 514}, {3: 1 << 31}, {4: -1}, {4: 65536}, {5: -1},
                                      {6: 7}, {6: 2048}, {6: 0}, {7: 0}, {7: 3}, {8: 80}, {9: None}, {12: None}, {14: None}, {14: P + 4},
                                      {15: None}, {15: P + 8}, {16: 0}, {13: -0.5}, {13: float("nan")}, {13: float("inf")},
                                      {11: P + 4}, {11: P, 5: 65}, {4: 60000, 5: 60000}] + [{12: c} for c in BAD_CACHE])
    refused("k2t_attn_tokens_workspace", [CTX, *shape, 8, C.byref(n)],
            [{0: None}, {1: -1}, {2: -1}, {3: 9}, {4: 0}, {5: 256}, {6: -1}, {6: (1 << 24) + 1}, {7: None}])
    if no_gpu():
        assert call("k2t_attn_tokens", *good) == HIP
        assert call("k2t_attn_tokens", CTX, 8, None, 512, 0, *shape[1:], None, None, None, rows(), 0.125, None, None, 0) == 0


@pytest.mark.parametrize("heads", [(32, 32, 64), (32, 8, 128), (32, 4, 128), (9, 3, 64), (40, 2, 64), (1, 1, 64)])
def test_attention_workspace_serves_less(heads):
    """The workspace of the largest block and longest cache is enough for a call with any smaller ones, and no
    less than theirs."""
    ctx = (C.c_int32 * 1024)(*[256] * 1024)  # a context of 256 CUs, on a device that no machine has

    def workspace(batch, ntok, length):
        n = C.c_size_t()
        assert call("k2t_attn_tokens_workspace", ctx, batch, ntok, *heads, length, C.byref(n)) == 0
        return n.value

    def accepted(batch, ntok, length, ws):
        rc = call("k2t_attn_tokens", ctx, 8, P, heads[0] * heads[2], batch, ntok, *heads, P, None, None,
                  rows(cap=1 << 24, length=length), 0.125, P, P, ws)
        assert rc in (-1, HIP)
        return rc == HIP

    lengths = [0, 1, 31, 64, 100, 127, 128, 129, 256, 300, 513, 1000, 1025, 2000, 2113, 4100, 4613, 9000, 12064, 65537, 1 << 20]
    for batch in (1, 3, 8):
        for ntok, length in [(64, 12064), (13, 2113), (515, 4613), (64, 300), (200, 1000), (8192, 8192), (33, 1 << 20), (1, 65537)]:
            ws = workspace(batch, ntok, length)
            for t in [x for x in (1, 2, 3, 5, 8, 10, 13, 16, 17, 24, 31, 32, 33, 48, 63, 64, 65, 100, 128, 200, 515, 3000, 8192) if x <= ntok]:
                for n in [x for x in lengths if x <= length]:
                    assert accepted(batch, t, n, ws), (batch, ntok, length, t, n)
                    assert workspace(batch, t, n) <= ws, (batch, ntok, length, t, n)


def rules(**change):
    r = k2t.LogitsRules()
    base = dict(history=P, history_len=P, prompt_len=P, repeat=P, presence=P, frequency=P, bias_tokens=P, bias=P, bias_len=P, mask=P,
                mask_row=P, history_stride=100, bias_stride=20, mask_stride=32, history_max=100, bias_max=20, mask_rows=4)
    for n, v in dict(base, **change).items():
        setattr(r, n, v)
    return r


def test_logits():
    keep = []

    def at(r):
        keep.append(r)
        return C.addressof(r)
    good = [CTX, P, 1000, 1000, 3, at(rules()), 2 * P, 1000]
    refused("k2t_logits_adjust", good, [{0: None}, {1: None}, {1: P + 2}, {2: 0}, {2: (1 << 24) + 1, 3: 1 << 25, 7: 1 << 25}, {3: 999}, {4: -1},
                                        {4: 65536}, {5: None}, {6: None}, {6: 2 * P + 1}, {7: 999}, {6: P, 7: 1004}, {3: 1 << 40}] +
            [{5: at(rules(**c))} for c in (dict(history=None), dict(history=None, repeat=None, presence=None), dict(history_stride=99),
                                           dict(history_max=-1), dict(history_max=(1 << 20) + 1, history_stride=1 << 21),
                                           dict(bias=None), dict(bias_tokens=None), dict(bias_stride=19), dict(bias_max=-1),
                                           dict(bias_max=4097, bias_stride=5000), dict(mask_stride=31), dict(mask_rows=-1),
                                           dict(mask_row=None, mask_rows=2), dict(mask=None))])
    if no_gpu():
        assert call("k2t_logits_adjust", *good) == HIP
        assert call("k2t_logits_adjust", CTX, None, 1000, 1000, 0, at(rules()), None, 1000) == 0
        assert call("k2t_logits_adjust", CTX, P, 1000, 1000, 3, at(rules(mask=None, mask_row=None)), P, 1000) == HIP


def test_keep():
    good = [CTX, 8, rows(), P, P, 5, None, 5, 2, 3, 2, 64]
    refused("k2t_kv_keep", good, [{0: None}, {1: 6}, {2: None}, {3: None}, {4: None}, {5: 4}, {5: 1 << 40}, {7: -1}, {7: (1 << 24) + 1, 5: 1 << 25},
                                  {8: -1}, {9: -1}, {9: 65536}, {10: 0}, {10: 1025}, {11: 32}, {8: 1 << 20, 9: 100},
                                  {8: 1 << 30, 9: 65535, 10: 1024}] + [{2: c} for c in BAD_CACHE])
    if no_gpu():
        assert call("k2t_kv_keep", *good) == HIP
        for nothing in (7, 8, 9):
            args = list(good)
            args[3] = args[4] = None
            args[nothing] = 0
            assert call("k2t_kv_keep", *args) == 0


def test_the_reference_itself():
    """block_ref on cases small enough to work out by hand."""
    x = np.zeros((1, 1, 4), np.float32)
    x[0, 0] = 1.0, 2.0, 3.0, 4.0
    quarter = np.array([0.25, 0.5], np.longdouble)  # one position: a quarter turn and half a turn
    y, _ = R.rope(x, np.array([1]), quarter, 1.0, False)
    assert np.allclose(y[0, 0], [-3.0, -2.0, 1.0, -4.0], atol=1e-15)
    y, _ = R.rope(x, np.array([1]), quarter, 2.0, True)
    assert np.allclose(y[0, 0], [-4.0, 2.0, -6.0, -8.0], atol=1e-14)
    assert R.visible(2, 1, 2, 4).tolist() == [[1, 1, 0, 0], [1, 1, 1, 0]]
    assert R.visible(2, 1, 1, 4, [3, 2]).tolist() == [[1, 1, 0, 0], [1, 0, 0, 0]]
    z = R.logits(np.array([[2.0, -2.0, 1.0, 5.0]], np.float32), 4,
                 dict(history=np.array([[0, 1, 1, 9]]), prompt_len=[1], repeat=[2.0], presence=[0.5], frequency=[0.25],
                      bias_tokens=np.array([[2, 2, -1]]), bias=np.array([[1.0, 2.0, 7.0]], np.float32), mask=np.array([[7]], np.int32)))
    assert z.tolist() == [[1.0, -5.0, 4.0, -np.inf]]
    a = np.arange(6).reshape(1, 1, 1, 6, 1)
    assert R.keep([a], [1], np.array([[0, 2, 1, 9]]), None, 4)[0].ravel().tolist() == [0, 1, 3, 3, 4, 5]


def test_logits_of_lists_without_entries():
    """A history that has no tokens yet, no biases, no masks this time: lists of length zero, which have no address."""
    import torch
    keep = []

    def at(r):
        keep.append(r)
        return C.addressof(r)
    good = [CTX, P, 1000, 1000, 3, at(rules(history=None, history_max=0, bias_tokens=None, bias=None, bias_max=0, mask=None, mask_rows=0)), 2 * P, 1000]
    refused("k2t_logits_adjust", good, [{5: at(rules(history=None, history_max=1))}, {5: at(rules(mask=None, mask_rows=1))},
                                        {5: at(rules(bias=None, bias_max=0))}])
    if no_gpu():
        assert call("k2t_logits_adjust", *good) == HIP
    i, f = dict(dtype=torch.int32), dict(dtype=torch.float32)
    for rows in (0, 3):
        r = k2t.LogitsRules(history=torch.zeros(rows, 0, **i), repeat=torch.ones(3, **f), bias_tokens=torch.zeros(rows, 0, **i),
                            bias=torch.zeros(rows, 0, **f), mask=torch.zeros(0, 40, **i), mask_row=torch.zeros(3, **i))
        assert (r.history, r.history_max, r.bias, r.bias_max, r.mask, r.mask_rows) == (None, 0, None, 0, None, 0) and r.repeat
    assert k2t.LogitsRules(history=torch.zeros(0, 5, **i)).history_max == 0
    with pytest.raises(ValueError):
        k2t.LogitsRules(mask=torch.zeros(3, 0, **i))


@pytest.mark.parametrize("heads", [(32, 32, 64), (32, 8, 128), (9, 3, 64), (16, 1, 128), (1, 1, 64)])
def test_attention_workspace_serves_fewer_rows(heads):
    """Requests of a batch that end leave fewer rows, whose positions are cut into more parts: the batch's workspace is
    enough for them."""
    ctx = (C.c_int32 * 1024)(*[256] * 1024)  # a context of 256 CUs, on a device that no machine has

    def workspace(batch, ntok, length):
        n = C.c_size_t()
        assert call("k2t_attn_tokens_workspace", ctx, batch, ntok, *heads, length, C.byref(n)) == 0
        return n.value

    for batch in (4, 16, 17, 64, 200):
        for ntok, length in [(1, 2000), (13, 2113), (64, 12064), (515, 4613), (40, 100)]:
            if batch * ntok * heads[0] > 1 << 22:
                continue
            ws = workspace(batch, ntok, length)
            for b in [x for x in (1, 2, 3, 5, 8, 11, 16, 31, 32, 33, 64, 100, 128, 199) if x < batch]:
                assert workspace(b, ntok, length) <= ws
                for t in {1, min(ntok, 16), ntok}:
                    for n in (1, 300, length):
                        rc = call("k2t_attn_tokens", ctx, 8, P, heads[0] * heads[2], b, t, *heads, P, None, None,
                                  rows(cap=1 << 24, length=min(n, length)), 0.125, P, P, ws)
                        assert rc == HIP, (batch, ntok, length, b, t, n)


def test_attention_workspace_of_no_rows():
    n = C.c_size_t()
    assert call("k2t_attn_tokens_workspace", CTX, 0, 2 ** 31 - 1, 16, 1, 64, 1 << 24, C.byref(n)) == 0 and n.value == 16
    assert call("k2t_attn_tokens_workspace", CTX, 5, 0, 16, 1, 64, 1 << 24, C.byref(n)) == 0 and n.value == 16
