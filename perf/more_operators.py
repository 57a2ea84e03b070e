"""Operators for blocks of tokens (prompts of a batch, drafted continuations), as measurable cases.

Four kinds, each through the public entry points of kronos-2t_amd/k2t.py:

  rope    rotary positions of the q and k heads of qkv rows: half or interleaved pairs, the whole head
          or part of it, frequencies scaled for long contexts, one position per token or drafted depths
  attn    attention of a block of tokens of every row over the row's Hadamard cache (int8 or NF4):
          causal for prompts, a visibility mask for trees of drafted tokens
  logits  penalties for repeated tokens, biases and grammar masks on rows of logits
  keep    the positions that a row keeps (the accepted path of a tree, what an eviction leaves) moved
          together in the caches of all layers, in place

run() computes a case in plain torch operations, or, where `own` is set, with the framework.
"""
import functools
import math
import os
import sys

import numpy as np
import torch

own = False
DEV = "cuda"
F32, F64 = torch.float32, torch.float64
# midpoints of the positive half of the NF4 codebook, and the codebook
NF4_CB = [-127, -96, -75, -58, -44, -31, -18, -6, 6, 18, 31, 44, 58, 75, 96, 127]
NF4_MID = [12.0, 24.5, 37.5, 51.0, 66.5, 85.5, 111.5]
FLT_EPS = 1.1920928955078125e-07


def listed():
    return [
        # one new token of four sequences in a 135M decoder's layer: the smallest call, latency alone
        dict(name="rope_one_token", kind="rope", batch=4, ntok=1, nq=9, nkv=3, hd=64, layout="half", rot=64,
             scaling="plain", start=700, ragged=False, tree=False),
        # a batch of prompts of different lengths, grouped heads, frequencies of a stretched context
        dict(name="rope_prompts", kind="rope", batch=6, ntok=777, nq=32, nkv=4, hd=128, layout="half", rot=128,
             scaling="ramp", start=100000, ragged=True, tree=False),
        # a 135M decoder checks ten drafted tokens behind a short prompt
        dict(name="attn_tree_short", kind="attn", bits=8, batch=1, ntok=10, nq=9, nkv=3, hd=64, start=300,
             ragged=False, tree=True),
        # eight requests check up to thirteen drafted tokens each over NF4 caches
        dict(name="attn_tree_requests_nf4", kind="attn", bits=4, batch=8, ntok=13, nq=32, nkv=8, hd=128, start=2100,
             ragged=True, tree=True),
        # a tree of sixty-four drafted tokens behind a long document
        dict(name="attn_tree_document", kind="attn", bits=8, batch=1, ntok=64, nq=32, nkv=4, hd=128, start=12000,
             ragged=False, tree=True),
        # a batch of prompts of a 1.7B decoder, plain heads, different lengths
        dict(name="attn_prompts", kind="attn", bits=8, batch=6, ntok=777, nq=32, nkv=32, hd=64, start=0,
             ragged=True, tree=False),
        # the next part of a prompt behind what an NF4 cache holds already
        dict(name="attn_prompt_part_nf4", kind="attn", bits=4, batch=1, ntok=515, nq=32, nkv=8, hd=128, start=4100,
             ragged=False, tree=False),
        # a long prompt at once, grouped heads: the largest
        dict(name="attn_prompt_long", kind="attn", bits=8, batch=1, ntok=8192, nq=32, nkv=4, hd=128, start=0,
             ragged=False, tree=False),
        # four requests, a hundred tokens of history, penalties alone
        dict(name="logits_small", kind="logits", rows=4, vocab=49152, history=100, bias=0, masked=False),
        # sixty-four requests over the largest vocabulary: long histories, biases, grammar states
        dict(name="logits_wide", kind="logits", rows=64, vocab=151936, history=2000, bias=40, masked=True),
        # four sequences of a 135M decoder keep the accepted path of ten drafted tokens, all layers
        dict(name="keep_accepted", kind="keep", bits=8, layers=30, rows=4, nkv=3, hd=64, start=300, length=10, keep=4),
        # three quarters of 4000 positions survive an eviction in a 1.7B decoder
        dict(name="keep_evicted", kind="keep", bits=8, layers=24, rows=1, nkv=32, hd=64, start=0, length=4000,
             keep=3000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(9, 3, 64), (32, 32, 64), (32, 4, 128), (32, 8, 128), (8, 2, 128), (16, 16, 128), (32, 4, 64)]


def draw(rng):
    kind = rng.choice(["rope", "attn", "attn", "attn", "logits", "keep"])
    nq, nkv, hd = rng.choice(HEADS)
    bits = rng.choice([8, 8, 4])
    if kind == "rope":
        batch, ntok = _log(rng, 1, 32), rng.choice([1, rng.randint(2, 64), _log(rng, 10, 1024)])
        while batch * ntok * (nq + nkv) * hd > 2.1e7:
            batch, ntok = max(1, batch * 2 // 3), max(1, ntok * 3 // 4)
        rot = rng.choice([hd, hd, hd // 2, 2 * rng.randint(1, hd // 2)])
        scaling = rng.choice(["plain", "linear", "base", "ramp", "wave"]) if rot >= 8 else "plain"
        return dict(kind=kind, batch=batch, ntok=ntok, nq=nq, nkv=nkv, hd=hd,
                    layout=rng.choice(["half", "half", "interleaved"]), rot=rot, scaling=scaling,
                    start=rng.choice([0, _log(rng, 1, 1000000)]), ragged=rng.random() < 0.5,
                    tree=ntok <= 64 and rng.random() < 0.5)
    if kind == "attn":
        tree = rng.random() < 0.5
        if tree:
            batch, ntok, start = _log(rng, 1, 16), _log(rng, 1, 64), _log(rng, 1, 16000)
        else:
            batch, ntok, start = _log(rng, 1, 16), _log(rng, 1, 8192), rng.choice([0, 0, _log(rng, 1, 8192)])
        while batch * ntok * (start + ntok / 2 + 20) * nq * hd > 1.3e11 or batch * (start + ntok) * nkv * hd > 1e8:
            batch, ntok, start = max(1, batch // 2), max(1, ntok * 3 // 4), start * 3 // 4
        return dict(kind=kind, bits=bits, batch=batch, ntok=ntok, nq=nq, nkv=nkv, hd=hd, start=start,
                    ragged=rng.random() < 0.5, tree=tree)
    if kind == "logits":
        rows, vocab = _log(rng, 1, 64), _log(rng, 1000, 151936)
        return dict(kind=kind, rows=rows, vocab=vocab, history=rng.choice([0, _log(rng, 1, 4000)]),
                    bias=rng.choice([0, _log(rng, 1, 300)]), masked=rng.random() < 0.5)
    layers, rows = rng.randint(1, 30), _log(rng, 1, 8)
    if rng.random() < 0.5:
        start, length = _log(rng, 1, 2000), _log(rng, 2, 64)
        keep = rng.randint(1, min(8, length))
    else:
        start, length = rng.choice([0, rng.randint(1, 16)]), _log(rng, 64, 8000)
        keep = max(1, int(length * rng.uniform(0.3, 0.95)))
    while layers * rows * nkv * hd * (start + length) > 1.5e8:
        layers, rows, start, length = max(1, layers // 2), max(1, rows // 2), start * 3 // 4, max(2, length * 3 // 4)
    return dict(kind=kind, bits=bits, layers=layers, rows=rows, nkv=nkv, hd=hd, start=start, length=length,
                keep=max(1, min(keep, length - 1)))


def work(case):
    kind = case["kind"]
    if kind == "logits":
        n = float(case["rows"]) * case["vocab"]
        return dict(bytes=8 * n + 4.0 * case["rows"] * case["history"] + (n / 8 if case["masked"] else 0.0), flops=2 * n)
    nkv, hd = case["nkv"], case["hd"]
    if kind == "rope":
        heads = case["batch"] * case["ntok"] * (case["nq"] + nkv) * (0.75 if case["ragged"] else 1.0)
        return dict(bytes=8.0 * heads * hd, flops=3.0 * heads * case["rot"])
    per = hd + 4 if case["bits"] == 8 else hd / 2 + hd / 32  # one quantized head and its scales
    if kind == "attn":
        b, nq = case["batch"], case["nq"]
        t = case["ntok"] * (0.75 if case["ragged"] else 1.0)
        start = case["start"] * (1.0 if b == 1 else 0.85)
        inside = min(t, 8.0) if case["tree"] else (t + 1) / 2  # (a drafted token's ancestors and itself)
        return dict(bytes=2.0 * nkv * per * b * (start + t) + 8.0 * b * t * nq * hd,
                    flops=4.0 * b * t * nq * hd * (start + inside))
    # (a position that stays where it is need not move: the leading ones of a path or an eviction hardly count)
    return dict(bytes=4.0 * case["layers"] * case["rows"] * nkv * case["keep"] * per, flops=0.0)


# ---------------------------------------------------------------- inputs
def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFF)


def _int(g, lo, hi, shape):
    return torch.randint(lo, hi, shape, generator=g, device=DEV, dtype=torch.int32)


def _counts(g, case, batch, ntok):
    if not case["ragged"]:
        return torch.full((batch,), ntok, dtype=torch.int32, device=DEV)
    return _int(g, (ntok + 1) // 2, ntok + 1, (batch,))


def _tree(seed, batch, ntok):
    """Drafted trees: every token hangs off one of the eight before it. Depths [batch][ntok], and which
    tokens of the block each one sees (its ancestors and itself) as the bits of int64."""
    rng = np.random.default_rng(int(seed) & 0x7FFFFFFF)
    depth, sees = np.zeros((batch, ntok), np.int32), np.zeros((batch, ntok), np.uint64)
    sees[:, 0] = 1
    at = np.arange(batch)
    for t in range(1, ntok):
        parent = t - 1 - rng.integers(0, min(8, t), batch)
        depth[:, t] = depth[at, parent] + 1
        sees[:, t] = sees[at, parent] | np.uint64(1 << t)
    return torch.from_numpy(depth).to(DEV), torch.from_numpy(sees.view(np.int64)).to(DEV)


def _rope_inputs(case, seed):
    g = _gen(seed, 1)
    b, t = case["batch"], case["ntok"]
    qkv = torch.randn(b * t, (case["nq"] + 2 * case["nkv"]) * case["hd"], generator=g, device=DEV)
    qkv[:, ::97] *= 8.0  # outlier channels, as projections have them
    pos = _int(g, 0, case["start"] + 1, (b,))
    depth = _tree(seed, b, t)[0] if case["tree"] else None
    return qkv, pos, _counts(g, case, b, t), depth


def _cache(g, bits, shape, hd):
    """K or V of `shape` slots: codes and scales as N(0, 1) heads quantize to."""
    x = torch.randn(*shape, hd, generator=g, device=DEV)
    if bits == 8:
        mx = x.abs().amax(-1, keepdim=True)
        return torch.round(x * (127.0 / mx)).to(torch.int8), (mx / 127.0).squeeze(-1)
    x = x.unflatten(-1, (-1, 64))
    mx = x.abs().amax(-1, keepdim=True)
    y = x * (127.0 / mx)
    p = torch.bucketize(y.abs(), torch.tensor(NF4_MID, device=DEV), right=True)
    idx = torch.where(y >= 0, 8 + p, 7 - p).to(torch.uint8).unflatten(-1, (2, 2, 16))
    return (idx[..., 0, :] | (idx[..., 1, :] << 4)).flatten(-3), (mx / 127.0).squeeze(-1).to(torch.bfloat16)


def _attn_inputs(case, seed):
    g = _gen(seed, 2)
    b, t, nkv, hd, bits = case["batch"], case["ntok"], case["nkv"], case["hd"], case["bits"]
    cap = case["start"] + t + 13
    q = 2.0 * torch.randn(b * t, case["nq"] * hd, generator=g, device=DEV)
    k, v = (_cache(g, bits, (b, nkv, cap), hd) for _ in range(2))
    pos = torch.full((b,), case["start"], dtype=torch.int32, device=DEV)
    if b > 1:  # sequences of different lengths
        pos = _int(g, int(0.7 * case["start"]), case["start"] + 1, (b,))
    sees = _tree(seed, b, t)[1] if case["tree"] else None
    return q, k, v, pos, _counts(g, case, b, t), sees


def _logits_inputs(case, seed):
    g = _gen(seed, 3)
    r, v, n, nb = case["rows"], case["vocab"], case["history"], case["bias"]
    d = dict(logits=3.0 * torch.randn(r, v, generator=g, device=DEV))
    if n:
        # common tokens come again and again
        d["history"] = (v * torch.rand(r, n, generator=g, device=DEV) ** 4).to(torch.int32).clamp(max=v - 1)
        d["history_len"] = _int(g, (n + 1) // 2, n + 1, (r,))
        d["prompt_len"] = _int(g, 0, n + 1, (r,))
        d["repeat"] = 1.0 + 0.3 * torch.rand(r, generator=g, device=DEV)
        d["presence"] = torch.rand(r, generator=g, device=DEV)
        d["frequency"] = 0.5 * torch.rand(r, generator=g, device=DEV)
    if nb:
        d["bias_tokens"] = _int(g, 0, v, (r, nb))
        d["bias"] = 5.0 * torch.randn(r, nb, generator=g, device=DEV)
        d["bias_len"] = _int(g, 0, nb + 1, (r,))
    if case["masked"]:
        # nine grammar states, from nearly everything allowed to few tokens; some rows have none
        share = torch.tensor([0.95, 0.9, 0.7, 0.5, 0.3, 0.1, 0.03, 0.01, 0.002], device=DEV)
        words = (v + 31) // 32
        bits = torch.rand(9, words, 32, generator=g, device=DEV) < share[:, None, None]
        weight = torch.tensor([1 << i for i in range(31)] + [-(1 << 31)], device=DEV, dtype=torch.int64)
        d["mask"] = (bits * weight).sum(-1).to(torch.int32)
        d["mask_row"] = _int(g, -1, 9, (r,))
    return d


def _keep_inputs(case, seed):
    g = _gen(seed, 4)
    n, rows, length, keep = case["layers"], case["rows"], case["length"], case["keep"]
    k, v = (_cache(g, case["bits"], (n, rows, case["nkv"], case["start"] + length), case["hd"]) for _ in range(2))
    pos = _int(g, 0, case["start"] + 1, (rows,))
    kept = torch.rand(rows, length, generator=g, device=DEV).argsort(-1)[:, :keep].sort(-1).values.to(torch.int32)
    return k, v, pos, kept.contiguous(), _int(g, (keep + 1) // 2, keep + 1, (rows,))


THETA, ORIGINAL, FACTOR = 100000.0, 8192, 16.0


def prepare(case, seed):
    kind = case["kind"]
    st = dict(case=case)
    if kind == "rope":
        st["x"], st["pos"], st["count"], st["depth"] = _rope_inputs(case, seed)
        st["out"] = torch.zeros_like(st["x"])
    elif kind == "attn":
        st["q"], st["k"], st["v"], st["pos"], st["count"], st["sees"] = _attn_inputs(case, seed)
        st["out"] = torch.zeros_like(st["q"])
    elif kind == "logits":
        st.update(_logits_inputs(case, seed))
        st["out"] = torch.zeros_like(st["logits"])
    else:
        st["k"], st["v"], st["pos"], st["kept"], st["count"] = _keep_inputs(case, seed)
    if own:
        _plan(st)
    elif kind == "rope":
        st["turns"], st["scale"] = _frequencies(case)
    elif kind != "logits":  # the rows' positions and tokens, as a host program has them
        st["host"] = list(zip(st["pos"].tolist(), st["count"].tolist()))
    return st


def _k2t():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kronos-2t_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import k2t
    return k2t


@functools.lru_cache(None)
def _context(stream):
    """A context whose calls run on `stream` (a stream's handle): a state's calls stay on the stream that
    was current when it was prepared, whatever is prepared after it."""
    ctx = _k2t().Ctx(0)
    ctx.set_stream(stream)
    return ctx


def _plan(st):
    """What a program keeps beside its data: the context, the caches' descriptions, plans and a workspace."""
    k2t, case, ctx = _k2t(), st["case"], _context(torch.cuda.current_stream().cuda_stream)
    st["ctx"] = ctx
    if case["kind"] == "rope":
        st["plan"] = k2t.RopePlan(layout={"half": k2t.ROPE_HALF, "interleaved": k2t.ROPE_INTERLEAVED}[case["layout"]],
                                  rot_dim=case["rot"], theta=THETA,
                                  scaling={"plain": k2t.ROPE_PLAIN, "linear": k2t.ROPE_LINEAR, "base": k2t.ROPE_BASE,
                                           "ramp": k2t.ROPE_RAMP, "wave": k2t.ROPE_WAVE}[case["scaling"]],
                                  factor=FACTOR, original=ORIGINAL)
    elif case["kind"] == "attn":
        cap = st["k"][0].shape[2]
        st["cache"] = k2t.KVRows(*st["k"], *st["v"], cap=cap, len=case["start"] + case["ntok"])
        ws = ctx.attn_tokens_workspace(case["batch"], case["ntok"], case["nq"], case["nkv"], case["hd"],
                                       case["start"] + case["ntok"])
        st["ws"] = torch.zeros(ws, dtype=torch.uint8, device=DEV)
    elif case["kind"] == "logits":
        names = ("history", "history_len", "prompt_len", "repeat", "presence", "frequency", "bias_tokens", "bias",
                 "bias_len", "mask", "mask_row")
        st["rules"] = k2t.LogitsRules(**{n: st[n] for n in names if n in st})
    else:
        st["cache"] = k2t.KVRows(*st["k"], *st["v"], cap=st["k"][0].shape[3])


# ---------------------------------------------------------------- one pass
def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if own:
        return {"rope": _own_rope, "attn": _own_attn, "logits": _own_logits, "keep": _own_keep}[kind](case, state)
    return {"rope": _plain_rope, "attn": _plain_attn, "logits": _plain_logits, "keep": _plain_keep}[kind](case, state)


def _own_rope(case, st):
    width = st["x"].shape[1]
    st["ctx"].rope(st["x"], width, case["batch"], case["ntok"], case["nq"] + case["nkv"], case["hd"], st["pos"],
                   st["plan"], st["out"], width, depth=st["depth"], counts=st["count"])
    return st["out"]


def _own_attn(case, st):
    st["ctx"].attn_tokens(case["bits"], st["q"], st["q"].shape[1], case["batch"], case["ntok"], case["nq"],
                          case["nkv"], case["hd"], st["pos"], st["cache"], case["hd"] ** -0.5, st["out"], st["ws"],
                          counts=st["count"], sees=st["sees"])
    return st["out"]


def _own_logits(case, st):
    v = case["vocab"]
    st["ctx"].logits_adjust(st["logits"], v, v, case["rows"], st["rules"], st["out"], v)
    return st["out"]


def _own_keep(case, st):
    st["ctx"].kv_keep(case["bits"], st["cache"], st["pos"], st["kept"], case["keep"], st["count"], case["keep"],
                      case["layers"], case["rows"], case["nkv"], case["hd"])
    return _flat(st)


def _flat(st):
    return dict(kq=st["k"][0], ks=st["k"][1], vq=st["v"][0], vs=st["v"][1])


# ---------------------------------------------------------------- the same in plain operations
def _frequencies(case):
    """Turns per position of every pair (fp64), and what the rotated values are multiplied by."""
    d, kind = case["rot"], case["scaling"]
    i = torch.arange(d // 2, dtype=F64, device=DEV)
    theta, scale = THETA, 1.0
    if kind == "base":
        theta = THETA * FACTOR ** (d / (d - 2))
    f = theta ** (-2.0 * i / d)
    if kind == "linear":
        f = f / FACTOR
    elif kind == "ramp":  # pairs that turn often stay, those that turn seldom are interpolated
        low, high = (d * math.log(ORIGINAL / (turns * 2 * math.pi)) / (2 * math.log(THETA)) for turns in (32.0, 1.0))
        low, high = max(math.floor(low), 0), min(math.ceil(high), d - 1)
        part = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f / FACTOR * part + f * (1 - part)
        scale = 0.1 * math.log(FACTOR) + 1.0
    elif kind == "wave":  # by wavelength: short ones stay, long ones are interpolated
        part = ((ORIGINAL * f / (2 * math.pi) - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        f = f / FACTOR * (1 - part) + f * part
    return f / (2 * math.pi), scale


def _pairs(case):
    half = torch.arange(case["rot"] // 2, device=DEV)
    return (half, half + case["rot"] // 2) if case["layout"] == "half" else (2 * half, 2 * half + 1)


def _plain_rope(case, st):
    b, t, heads, hd, rot = case["batch"], case["ntok"], case["nq"] + case["nkv"], case["hd"], case["rot"]
    step = torch.arange(t, device=DEV)
    pos = st["pos"][:, None] + (st["depth"] if st["depth"] is not None else step)  # [b][t]
    turn = pos.to(F64)[..., None] * st["turns"]
    angle = (turn - torch.round(turn)) * (2 * math.pi)  # [b][t][pairs]
    cos, sin = ((f(angle) * st["scale"]).to(F32)[:, :, None] for f in (torch.cos, torch.sin))
    x = st["x"].view(b, t, -1, hd)
    out = st["out"].view(b, t, -1, hd)
    y = x[:, :, :heads].clone()
    lo, hi = _pairs(case)
    x0, x1 = x[:, :, :heads, lo], x[:, :, :heads, hi]
    y[..., lo], y[..., hi] = x0 * cos - x1 * sin, x1 * cos + x0 * sin
    here = (step < st["count"][:, None])[..., None, None]
    out[:, :, :heads] = torch.where(here, y, out[:, :, :heads])
    return st["out"]


def _signs(block):
    """Sign of each element of Hadamard block `block` (SplitMix64 of the block's seed)."""
    mask, out = (1 << 64) - 1, []
    for i in range(64):
        z = (0x9E3779B97F4A7C15 + block * 0xBF58476D1CE4E5B9 + (i + 1) * 0x9E3779B97F4A7C15) & mask
        z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & mask
        z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & mask
        out.append(-1.0 if (z ^ (z >> 31)) & 1 else 1.0)
    return out


@functools.lru_cache(None)
def _sign_rows(blocks, dtype, dev):
    return torch.tensor([_signs(b) for b in range(blocks)], dtype=dtype, device=dev)


def _stage(v, h):
    a = v.unflatten(-1, (-1, 2, h))
    x, y = a[..., 0, :], a[..., 1, :]
    return torch.stack((x + y, x - y), -2).flatten(-3)


def _butterflies(v):
    """H64 of the last dimension, in the order that the cache's format fixes."""
    return functools.reduce(_stage, (1, 2, 4, 8, 16, 32), v)


def _rotate(x):
    """Signed Hadamard-64 of the last dimension's blocks; [..., blocks, 64]."""
    v = x.unflatten(-1, (-1, 64))
    return _butterflies(v * (0.125 * _sign_rows(v.shape[-2], F32, str(x.device))))


def _unrotate(v):
    return (_butterflies(v) * (0.125 * _sign_rows(v.shape[-2], F32, str(v.device)))).flatten(-2)


def _quant8(r):
    """int8 codes and the scale of rotated heads [..., blocks, 64]."""
    mx = r.abs().amax((-2, -1), keepdims=True)
    small = mx <= FLT_EPS
    q = torch.round(r * (torch.full_like(mx, 127.0) / mx))  # (one rounding: a scalar over a tensor has two)
    q, s = torch.where(small, torch.zeros_like(q), q), torch.where(small, torch.zeros_like(mx), mx / 127.0)
    return q.flatten(-2), s[..., 0, 0]


def _values(codes, scales, bits, dtype=F32):
    """Rotated heads [..., hd] that a cache's codes and scales stand for."""
    if bits == 8:
        return codes.to(dtype) * scales.to(dtype)[..., None]
    cb = torch.tensor(NF4_CB, dtype=dtype, device=codes.device)
    b = codes.unflatten(-1, (-1, 2, 16))
    idx = torch.stack((b & 15, b >> 4), -2).flatten(-3)  # [..., blocks, 64]
    return (cb[idx.to(torch.int64)] * scales.to(dtype)[..., None]).flatten(-2)


def _visible(case, sees, count, start, row, n):
    """Whether each token of a row [ntok] sees position [n] of its cache."""
    step, at = torch.arange(case["ntok"], device=DEV)[:, None], torch.arange(n, device=DEV)[None, :] - start
    if sees is None:
        return at <= step
    bit = (sees[row][:, None] >> at.clamp(0, 63)) & 1
    return (at < 0) | ((bit != 0) & (at < count))


def _plain_attn(case, st):
    b, t, nq, nkv, hd, bits = (case[x] for x in ("batch", "ntok", "nq", "nkv", "hd", "bits"))
    g = nq // nkv
    q, qs = _quant8(_rotate(st["q"].view(b, t, nkv, g, hd)))
    qs = qs * (hd ** -0.5)
    out = st["out"].view(b, t, nkv, g, hd)
    for row, (start, count) in enumerate(st["host"]):
        n = start + count
        hidden = ~_visible(case, st["sees"], count, start, row, n)[:count, None, :]
        for h in range(nkv):
            k, ks, v, vs = st["k"][0][row, h, :n], st["k"][1][row, h, :n], st["v"][0][row, h, :n], st["v"][1][row, h, :n]
            codes, scale = q[row, :count, h], qs[row, :count, h, :, None]  # [count][g][hd]
            if bits == 8:  # whole products below 2^24: the sums are exact
                z = (codes @ k.to(F32).T) * ks * scale
            else:
                z = (codes @ _values(k, ks, bits).T) * scale
            z = z.masked_fill(hidden, -math.inf)
            p = torch.exp(z - z.amax(-1, keepdim=True))
            o = (p @ _values(v, vs, bits)) / p.sum(-1, keepdim=True)
            out[row, :count, h] = _unrotate(o.unflatten(-1, (-1, 64)))
    return st["out"]


def _listed_counts(tokens, live, v):
    """How often each token of the vocabulary stands in rows of tokens where `live`."""
    out = torch.zeros(tokens.shape[0], v, dtype=torch.int32, device=DEV)
    return out.scatter_add_(1, tokens.long(), live.to(torch.int32))


def _plain_logits(case, st):
    v = case["vocab"]
    x = st["logits"].to(F64)  # (differences of large penalties: rounded once at the end)
    col = lambda n: st[n].to(F64)[:, None]  # noqa: E731
    if case["history"]:
        step = torch.arange(case["history"], device=DEV)
        live = step < st["history_len"][:, None]
        seen = _listed_counts(st["history"], live, v) > 0
        fresh = _listed_counts(st["history"], live & (step >= st["prompt_len"][:, None]), v).to(F64)
        x = torch.where(seen, torch.where(x > 0, x / col("repeat"), x * col("repeat")), x)
        x = x - col("frequency") * fresh - col("presence") * (fresh > 0)
    if case["bias"]:
        live = torch.arange(case["bias"], device=DEV) < st["bias_len"][:, None]
        add = torch.where(live, st["bias"], torch.zeros_like(st["bias"])).to(F64)
        x = x.scatter_add(1, st["bias_tokens"].long(), add)
    if case["masked"]:
        row = st["mask_row"].long()
        token = torch.arange(v, device=DEV)
        allowed = (st["mask"][row.clamp(min=0)][:, token // 32] >> (token % 32)) & 1
        x = torch.where((row[:, None] >= 0) & (allowed == 0), torch.full_like(x, -math.inf), x)
    st["out"].copy_(x)
    return st["out"]


def _plain_keep(case, st):
    for x in (*st["k"], *st["v"]):
        for row, (start, count) in enumerate(st["host"]):
            x[:, row, :, start:start + count] = x[:, row][:, :, start + st["kept"][row, :count].long()]
    return _flat(st)


# ---------------------------------------------------------------- the same in 64 bits
def _hadamard():
    i = np.arange(64)
    return 1.0 - 2.0 * (np.array([bin(a).count("1") for a in range(64)])[i[:, None] & i[None, :]] & 1)


def _codes(x):
    """int8 codes and scales of heads x [..., hd] (numpy fp32): the format's own fp32 arithmetic, which
    codes next to a border depend on."""
    f = np.float32
    v = x.reshape(x.shape[:-1] + (-1, 64)) * np.array([_signs(b) for b in range(x.shape[-1] // 64)], f) * f(0.125)
    for h in (1, 2, 4, 8, 16, 32):
        low = (np.arange(64) & h) == 0
        a, b = v[..., low], v[..., ~low]
        v = np.empty_like(v)
        v[..., low], v[..., ~low] = a + b, a - b
    mx = np.abs(v).max((-2, -1), keepdims=True)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(mx <= FLT_EPS, f(0), np.rint(v * (f(127.0) / mx)))
    return q.reshape(x.shape).astype(np.int8), np.where(mx <= FLT_EPS, f(0), mx / f(127.0))[..., 0]


def _unrot64(v):
    """Inverse rotation of [..., blocks, 64] in 64 bits, on the GPU."""
    h = torch.from_numpy(_hadamard()).to(v.device) / 8.0
    return ((v @ h) * _sign_rows(v.shape[-2], F64, str(v.device))).flatten(-2)


def _exact_rope(case, seed):
    x, pos, count, depth = _rope_inputs(case, seed)
    b, t, heads, hd, d = case["batch"], case["ntok"], case["nq"] + case["nkv"], case["hd"], case["rot"]
    n = d // 2
    # the angles in units of a turn, as numpy's long double
    ld = np.longdouble
    i, two_pi = np.arange(n, dtype=ld), 2 * ld(np.pi) + ld(2.4492935982947064e-16)
    theta = ld(THETA) * ld(FACTOR) ** (ld(d) / (d - 2)) if case["scaling"] == "base" else ld(THETA)
    f = theta ** (-2 * i / d)
    factor = 1.0
    if case["scaling"] == "linear":
        f = f / ld(FACTOR)
    elif case["scaling"] == "ramp":
        edge = [d * math.log(ORIGINAL / (r * 2 * math.pi)) / (2 * math.log(THETA)) for r in (32.0, 1.0)]
        lo, hi = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), d - 1)
        w = np.clip((i - lo) / ld(max(hi - lo, 0.001)), 0, 1)
        f = f * (1 - w) + f / ld(FACTOR) * w
        factor = 1.0 + 0.1 * math.log(FACTOR)
    elif case["scaling"] == "wave":
        w = np.clip((ORIGINAL / (two_pi / f) - 1) / 3, 0, 1)
        f = f * w + f / ld(FACTOR) * (1 - w)
    at = pos.cpu().numpy().astype(np.int64)[:, None] + (np.arange(t) if depth is None else depth.cpu().numpy())
    turn = at.astype(ld)[..., None] * (f / two_pi)
    turn = torch.from_numpy((turn - np.rint(turn)).astype(np.float64)).to(DEV) * (2 * math.pi)
    rot = torch.polar(torch.full_like(turn, factor), turn)[:, :, None]  # [b][t][1][pairs]
    v = x.view(b, t, -1, hd)[:, :, :heads].to(F64)
    out = torch.zeros(b, t, x.shape[1] // hd, hd, dtype=F64, device=DEV)
    out[:, :, :heads] = v
    if case["layout"] == "half":
        z = torch.complex(v[..., :n], v[..., n:d]) * rot
        out[:, :, :heads, :n], out[:, :, :heads, n:d] = z.real, z.imag
    else:
        z = torch.complex(v[..., 0:d:2], v[..., 1:d:2]) * rot
        out[:, :, :heads, 0:d:2], out[:, :, :heads, 1:d:2] = z.real, z.imag
    out[torch.arange(t, device=DEV) >= count[:, None]] = 0.0
    return out.view(b * t, -1)


def _exact_attn(case, seed):
    q, k, v, pos, count, sees = _attn_inputs(case, seed)
    b, t, nq, nkv, hd, bits = (case[x] for x in ("batch", "ntok", "nq", "nkv", "hd", "bits"))
    code, qs = _codes(q.cpu().numpy().reshape(b, t, nkv, nq // nkv, hd))
    code, qs = torch.from_numpy(code).to(DEV), torch.from_numpy(qs).to(DEV)
    out = torch.zeros(b, t, nkv, nq // nkv, hd, dtype=F64, device=DEV)
    for row in range(b):
        start, n = int(pos[row]), int(count[row])
        hidden = ~_visible(case, sees, n, start, row, start + n)
        for h in range(nkv):
            kk, vv = (_values(c[row, h, :start + n], s[row, h, :start + n], bits, F64) for c, s in (k, v))
            for a in range(0, n, 1024):  # (a part of the tokens at a time)
                z = min(a + 1024, n)
                qv = code[row, a:z, h].to(F64) * (qs[row, a:z, h].to(F64) / math.sqrt(hd))
                s = (qv @ kk.T).masked_fill(hidden[a:z, None], -math.inf)
                out[row, a:z, h] = torch.softmax(s, -1) @ vv
    return _unrot64(out.unflatten(-1, (-1, 64))).reshape(b * t, nq * hd)


def _exact_logits(case, seed):
    d = _logits_inputs(case, seed)
    out = d["logits"].to(F64)
    x = out.cpu().numpy()
    host = {n: a.cpu().numpy() for n, a in d.items() if n != "logits"}
    for r in range(case["rows"]):
        if case["history"]:
            past = host["history"][r, :host["history_len"][r]]
            seen = np.unique(past)
            rep = np.float64(host["repeat"][r])
            x[r, seen] = np.where(x[r, seen] > 0, x[r, seen] / rep, x[r, seen] * rep)
            token, times = np.unique(past[host["prompt_len"][r]:], return_counts=True)
            x[r, token] -= np.float64(host["presence"][r]) + np.float64(host["frequency"][r]) * times
        for i in range(int(host["bias_len"][r]) if case["bias"] else 0):
            x[r, host["bias_tokens"][r, i]] += np.float64(host["bias"][r, i])
        if case["masked"] and host["mask_row"][r] >= 0:
            bits = np.unpackbits(host["mask"][host["mask_row"][r]].view(np.uint8), bitorder="little")[:case["vocab"]]
            x[r, bits == 0] = -np.inf
    return torch.from_numpy(x).to(DEV)


def _exact_keep(case, seed):
    k, v, pos, kept, count = _keep_inputs(case, seed)
    out = {}
    for name, (_, scales) in (("k", k), ("v", v)):
        new = scales.to(F64)
        for row in range(case["rows"]):
            p, n = int(pos[row]), int(count[row])
            new[:, row, :, p:p + n] = scales[:, row][:, :, (p + kept[row, :n]).long()].to(F64)
        out[name + "s"] = new
    return dict(kq=None, ks=out["ks"], vq=None, vs=out["vs"])


def exact(case, seed):
    return {"rope": _exact_rope, "attn": _exact_attn, "logits": _exact_logits, "keep": _exact_keep}[case["kind"]](case, seed)
