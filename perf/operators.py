"""Operators for several continuations of one prompt, as measurable cases.

Four kinds, each through the public entry points of kronos-2t_amd/k2t.py:

  kv       heads of a batch of sequences quantized into a Hadamard cache (int8 or NF4) at each
           sequence's position, and the same positions read back as fp32 heads
  attn     one token's attention for rows (beams, samples) that share their sequence's prefix
           cache and have a tail cache each
  select   the best k continuations of every sequence over its beams and the vocabulary
  reorder  the tail caches of all layers rearranged to the chosen beams, in place

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
FLT_EPS, FLT_MAX = 1.1920928955078125e-07, 3.4028234663852886e38


def listed():
    return [
        # one new token of four beams in a 135M decoder's layer: the smallest call, latency alone
        dict(name="kv_one_token", kind="kv", bits=8, batch=4, ntok=1, nkv=3, nq=9, hd=64, start=40, ragged=False),
        # a batch of prompts of different lengths, up to 777 tokens, into an int8 cache
        dict(name="kv_prompts", kind="kv", bits=8, batch=6, ntok=777, nkv=4, nq=32, hd=128, start=0, ragged=True),
        # a prompt of plain heads into the compact NF4 cache, behind 100 cached positions
        dict(name="kv_prompt_nf4", kind="kv", bits=4, batch=1, ntok=515, nkv=32, nq=32, hd=64, start=100,
             ragged=False),
        # four beams over a short prompt of a 135M decoder
        dict(name="attn_short", kind="attn", bits=8, n_seq=1, beams=4, nq=9, nkv=3, hd=64, prefix=45, tail=7),
        # eight beams of a 1.7B decoder, plain heads, a prompt of ordinary length
        dict(name="attn_mha", kind="attn", bits=8, n_seq=1, beams=8, nq=32, nkv=32, hd=64, prefix=1500, tail=64),
        # three requests of eight beams each over the NF4 cache, prompts of different lengths
        dict(name="attn_nf4_requests", kind="attn", bits=4, n_seq=3, beams=8, nq=32, nkv=8, hd=128, prefix=4100,
             tail=90),
        # sixty-four samples of one long document question, grouped heads: the largest
        dict(name="attn_many_samples", kind="attn", bits=8, n_seq=1, beams=64, nq=32, nkv=4, hd=128, prefix=12000,
             tail=333),
        # four beams over a small vocabulary
        dict(name="select_small", kind="select", n_seq=1, beams=4, vocab=8192, k=4, done=False, banned=False),
        # eight requests of eight beams, twice as many candidates as beams, some tokens ruled out
        dict(name="select_requests", kind="select", n_seq=8, beams=8, vocab=49152, k=16, done=True, banned=True),
        # sixteen beams over the largest vocabulary
        dict(name="select_wide", kind="select", n_seq=1, beams=16, vocab=151936, k=32, done=False, banned=False),
        # four beams of a 135M decoder a few tokens in
        dict(name="reorder_135m", kind="reorder", bits=8, layers=30, n_seq=1, beams=4, nkv=3, hd=64, cap=64, len=21),
        # eight beams of a 1.7B decoder two hundred tokens in
        dict(name="reorder_1.7b", kind="reorder", bits=8, layers=24, n_seq=1, beams=8, nkv=32, hd=64, cap=256,
             len=200),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(9, 3, 64), (32, 32, 64), (32, 4, 128), (32, 8, 128), (8, 2, 128), (16, 16, 128)]


def draw(rng):
    kind = rng.choice(["kv", "attn", "attn", "select", "reorder"])
    nq, nkv, hd = rng.choice(HEADS)
    bits = rng.choice([8, 8, 4])
    if kind == "kv":
        batch = _log(rng, 1, 32)
        ntok = rng.choice([1, rng.randint(2, 9), _log(rng, 10, 1024)])
        while batch * ntok * nkv * hd > 2.3e6:
            batch, ntok = max(1, batch * 2 // 3), max(1, ntok * 3 // 4)
        return dict(kind=kind, bits=bits, batch=batch, ntok=ntok, nkv=nkv, nq=nq, hd=hd,
                    start=rng.choice([0, _log(rng, 1, 500)]), ragged=rng.random() < 0.5)
    if kind == "attn":
        n_seq = rng.choice([1, 1, 1, 2, 4])
        beams = _log(rng, 1, 64 // n_seq)
        return dict(kind=kind, bits=bits, n_seq=n_seq, beams=beams, nq=nq, nkv=nkv, hd=hd,
                    prefix=_log(rng, 16, 12000 // n_seq), tail=_log(rng, 1, 333))
    if kind == "select":
        n_seq, beams = _log(rng, 1, 8), _log(rng, 1, 32)
        vocab = _log(rng, 1000, 151936)
        while n_seq * beams * vocab > 3.1e6:
            n_seq, vocab = max(1, n_seq // 2), max(1000, vocab * 2 // 3)
        return dict(kind=kind, n_seq=n_seq, beams=beams, vocab=vocab, k=rng.choice([beams, 2 * beams]),
                    done=rng.random() < 0.5, banned=rng.random() < 0.5)
    layers, n_seq, beams, length = rng.randint(1, 30), rng.choice([1, 1, 2, 5]), rng.randint(2, 16), _log(rng, 1, 400)
    while layers * n_seq * beams * nkv * hd * length > 7.5e7:
        layers, length = max(1, layers // 2), max(1, length * 3 // 4)
    return dict(kind=kind, bits=bits, layers=layers, n_seq=n_seq, beams=beams, nkv=nkv, hd=hd,
                cap=length + rng.randint(0, 100), len=length)


def work(case):
    if case["kind"] == "select":
        n = case["n_seq"] * case["beams"] * case["vocab"]
        return dict(bytes=4.0 * n + 8 * case["n_seq"] * (case["beams"] + 2 * case["k"]), flops=4.0 * n)
    nkv, hd = case["nkv"], case["hd"]
    per = hd + 4 if case["bits"] == 8 else hd / 2 + hd / 32  # one quantized head and its scales
    if case["kind"] == "kv":
        heads = 2.0 * case["batch"] * case["ntok"] * nkv * (0.75 if case["ragged"] else 1.0)
        return dict(bytes=2 * heads * (4 * hd + per), flops=2 * heads * hd * 10)
    if case["kind"] == "attn":
        rows, nq = case["n_seq"] * case["beams"], case["nq"]
        pre = case["prefix"] * (1.0 if case["n_seq"] == 1 else 0.85)
        tail = case["tail"] * 0.85
        return dict(bytes=2 * nkv * per * (case["n_seq"] * pre + rows * tail) + 8.0 * rows * nq * hd,
                    flops=4.0 * rows * nq * hd * (pre + tail))
    b = case["beams"]  # parents drawn with replacement: rows that move, and distinct sources
    moved = b - 1 + b * (1 - (1 - 1 / b) ** b)
    return dict(bytes=case["layers"] * case["n_seq"] * moved * nkv * case["len"] * 2.0 * per, flops=0.0)


# ---------------------------------------------------------------- inputs
def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFF)


def _int(g, lo, hi, shape):
    return torch.randint(lo, hi, shape, generator=g, device=DEV, dtype=torch.int32)


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


def _kv_inputs(case, seed):
    g = _gen(seed, 1)
    b, t, nkv, hd = case["batch"], case["ntok"], case["nkv"], case["hd"]
    qkv = torch.randn(b * t, (case["nq"] + 2 * nkv) * hd, generator=g, device=DEV)
    qkv[:, ::97] *= 8.0  # outlier channels, as projections have them
    pos = _int(g, 0, case["start"] + 1, (b,))
    count = _int(g, (t + 1) // 2, t + 1, (b,)) if case["ragged"] else torch.full((b,), t, dtype=torch.int32, device=DEV)
    return qkv, pos, count


def _attn_inputs(case, seed):
    g = _gen(seed, 2)
    n_seq, beams, nkv, hd, bits = case["n_seq"], case["beams"], case["nkv"], case["hd"], case["bits"]
    pcap, tcap, rows = case["prefix"] + 13, case["tail"] + 5, n_seq * beams
    q = 2.0 * torch.randn(rows, case["nq"] * hd, generator=g, device=DEV)
    pk, pv = (_cache(g, bits, (n_seq, nkv, pcap), hd) for _ in range(2))
    tk, tv = (_cache(g, bits, (rows, nkv, tcap), hd) for _ in range(2))
    plen = torch.full((n_seq,), case["prefix"], dtype=torch.int32, device=DEV)
    if n_seq > 1:  # prompts of different lengths
        plen = _int(g, int(0.7 * case["prefix"]), case["prefix"] + 1, (n_seq,))
    # beams of one sequence are equally long but for those that have ended
    tlen = _int(g, int(0.7 * case["tail"]), case["tail"] + 1, (rows,))
    return q, pk, pv, tk, tv, plen, tlen


def _select_inputs(case, seed):
    g = _gen(seed, 3)
    n, beams, v = case["n_seq"], case["beams"], case["vocab"]
    logits = 3.0 * torch.randn(n * beams, v, generator=g, device=DEV)
    if case["banned"]:
        logits[:, torch.randperm(v, generator=g, device=DEV)[:v // 10]] = -math.inf
    scores = -2.0 * torch.rand(n * beams, generator=g, device=DEV) - 3.0
    done = torch.zeros(n * beams, dtype=torch.int32, device=DEV)
    if case["done"]:
        done = (torch.rand(n * beams, generator=g, device=DEV) < 0.2).to(torch.int32)
    return logits, scores, done


def _reorder_inputs(case, seed):
    g = _gen(seed, 4)
    n, beams = case["n_seq"], case["beams"]
    shape = (case["layers"], n * beams, case["nkv"], case["cap"])
    k, v = (_cache(g, case["bits"], shape, case["hd"]) for _ in range(2))
    base = torch.arange(n, dtype=torch.int32, device=DEV).repeat_interleave(beams) * beams
    parents = base + _int(g, 0, beams, (n * beams,))
    return k, v, parents


def prepare(case, seed):
    kind = case["kind"]
    st = dict(case=case)
    if kind == "kv":
        st["qkv"], st["pos"], st["count"] = _kv_inputs(case, seed)
        # (one slot more than any sequence needs)
        hd, cap = case["hd"], case["start"] + case["ntok"] + 1
        slots = (case["batch"], case["nkv"], cap)
        codes, scale = ((hd,), F32) if case["bits"] == 8 else ((hd // 2,), torch.bfloat16)
        for n in "kv":
            st[n + "q"] = torch.zeros(slots + codes, dtype=torch.int8 if case["bits"] == 8 else torch.uint8, device=DEV)
            st[n + "s"] = torch.zeros(slots + (() if case["bits"] == 8 else (hd // 64,)), dtype=scale, device=DEV)
            st[n] = torch.zeros(case["batch"] * case["ntok"], case["nkv"] * hd, device=DEV)
    elif kind == "attn":
        q, pk, pv, tk, tv, plen, tlen = _attn_inputs(case, seed)
        st.update(q=q, pk=pk, pv=pv, tk=tk, tv=tv, plen=plen, tlen=tlen, out=torch.zeros_like(q))
    elif kind == "select":
        st["logits"], st["scores"], st["done"] = _select_inputs(case, seed)
        st["eos"] = 2
        n = (case["n_seq"], case["k"])
        st["out"] = dict(scores=torch.zeros(n, device=DEV),
                         **{x: torch.zeros(n, dtype=torch.int32, device=DEV) for x in ("tokens", "parents", "done")})
    else:
        st["k"], st["v"], st["parents"] = _reorder_inputs(case, seed)
        st["len"] = torch.full_like(st["parents"], case["len"])
    if own:
        _plan(st)
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
    """What a program keeps beside its data: the context, the caches' descriptions and a workspace."""
    k2t, case, ctx = _k2t(), st["case"], _context(torch.cuda.current_stream().cuda_stream)
    st["ctx"], ws = ctx, 0
    if case["kind"] == "kv":
        st["cache"] = k2t.KVRows(st["kq"], st["ks"], st["vq"], st["vs"], cap=st["kq"].shape[2])
    elif case["kind"] == "attn":
        st["prefix"] = k2t.KVRows(*st["pk"], *st["pv"], cap=st["pk"][0].shape[2], len=case["prefix"], d_len=st["plen"])
        st["tail"] = k2t.KVRows(*st["tk"], *st["tv"], cap=st["tk"][0].shape[2], len=case["tail"], d_len=st["tlen"])
        ws = ctx.attn_shared_workspace(case["n_seq"], case["beams"], case["nq"], case["nkv"], case["hd"],
                                       case["prefix"], case["tail"])
    elif case["kind"] == "select":
        ws = ctx.beam_select_workspace(case["n_seq"], case["beams"], case["vocab"], case["k"])
    else:
        st["cache"] = k2t.KVRows(*st["k"], *st["v"], cap=case["cap"], len=case["len"], d_len=st["len"])
    st["ws"] = torch.zeros(ws, dtype=torch.uint8, device=DEV)


# ---------------------------------------------------------------- one pass
def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if own:
        return {"kv": _own_kv, "attn": _own_attn, "select": _own_select, "reorder": _own_reorder}[kind](case, state)
    return {"kv": _plain_kv, "attn": _plain_attn, "select": _plain_select, "reorder": _plain_reorder}[kind](case, state)


def _own_kv(case, st):
    ctx, hd, nkv = st["ctx"], case["hd"], case["nkv"]
    width = st["qkv"].shape[1]
    k = st["qkv"].data_ptr() + 4 * case["nq"] * hd  # the k heads of a qkv row, then its v heads
    v = k + 4 * nkv * hd
    ctx.kv_append(case["bits"], k, v, width, case["batch"], case["ntok"], nkv, hd, st["pos"], st["cache"],
                  counts=st["count"])
    ctx.kv_load(case["bits"], st["cache"], case["batch"], case["ntok"], nkv, hd, st["pos"], st["k"], st["v"],
                nkv * hd, counts=st["count"])
    return dict(k=st["k"], v=st["v"])


def _own_attn(case, st):
    st["ctx"].attn_shared(case["bits"], st["q"], st["q"].shape[1], case["n_seq"], case["beams"], case["nq"],
                          case["nkv"], case["hd"], st["prefix"], st["tail"], case["hd"] ** -0.5, st["out"], st["ws"])
    return st["out"]


def _own_select(case, st):
    o = st["out"]
    st["ctx"].beam_select(st["logits"], case["vocab"], case["vocab"], st["scores"], st["done"], case["n_seq"],
                          case["beams"], case["k"], st["eos"], o["scores"], o["tokens"], o["parents"], o["done"],
                          st["ws"])
    return o


def _own_reorder(case, st):
    st["ctx"].kv_reorder(case["bits"], st["cache"], st["parents"], case["layers"], case["n_seq"], case["beams"],
                         case["nkv"], case["hd"])
    return _flat(st)


def _flat(st):
    return dict(kq=st["k"][0], ks=st["k"][1], vq=st["v"][0], vs=st["v"][1])


# ---------------------------------------------------------------- the same in plain operations
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
    mx = r.abs().amax((-2, -1), keepdim=True)
    small = mx <= FLT_EPS
    q = torch.round(r * (torch.full_like(mx, 127.0) / mx))  # (one rounding: a scalar over a tensor has two)
    q, s = torch.where(small, torch.zeros_like(q), q), torch.where(small, torch.zeros_like(mx), mx / 127.0)
    return q.flatten(-2), s[..., 0, 0]


def _nf4_index(y):
    p = torch.bucketize(y.abs(), torch.tensor(NF4_MID, device=y.device), right=True)
    return torch.where(y >= 0, 8 + p, 7 - p)


def _quant4(r):
    """NF4 bytes and BF16 block scales of rotated heads [..., blocks, 64]."""
    cb = torch.tensor(NF4_CB, dtype=F32, device=r.device)
    mx = r.abs().amax(-1, keepdim=True)
    c = cb[_nf4_index(r * (torch.full_like(mx, 127.0) / mx))]
    # sums in element order, which decides the scale's last bit: a running sum down a leading dimension
    num = torch.cumsum((r * c).movedim(-1, 0), 0)[-1].unsqueeze(-1)
    den = (c * c).sum(-1, keepdim=True)
    s = torch.where((den > 1e-12) & (num > 0), num / den, mx / 127.0)
    small = mx < 1e-30
    s = torch.where(small, torch.zeros_like(s), s).to(torch.bfloat16)
    inv = torch.where(s > 1e-30, 1.0 / s.to(F32), torch.zeros_like(mx))
    idx = torch.where(small, torch.full_like(r, 8, dtype=torch.int64), _nf4_index(r * inv))
    idx = idx.to(torch.uint8).unflatten(-1, (2, 2, 16))
    return (idx[..., 0, :] | (idx[..., 1, :] << 4)).flatten(-3), s.squeeze(-1)


def _values(codes, scales, bits, dtype=F32):
    """Rotated heads [..., blocks, 64] that a cache's codes and scales stand for."""
    if bits == 8:
        return codes.to(dtype).unflatten(-1, (-1, 64)) * scales.to(dtype)[..., None, None]
    cb = torch.tensor(NF4_CB, dtype=dtype, device=codes.device)
    b = codes.unflatten(-1, (-1, 2, 16))
    idx = torch.stack((b & 15, b >> 4), -2).flatten(-3)  # [..., blocks, 64]
    return cb[idx.to(torch.int64)] * scales.to(dtype)[..., None]


def _plain_kv(case, st):
    b, t, nq, nkv, hd = (case[x] for x in ("batch", "ntok", "nq", "nkv", "hd"))
    step = torch.arange(t, device=st["pos"].device)
    here = step < st["count"][:, None]  # [batch][ntok]
    # tokens that a shorter sequence does not have go to the spare last slot
    slot = torch.where(here, st["pos"][:, None] + step, st["kq"].shape[2] - 1).long()
    row, head = torch.arange(b, device=slot.device)[:, None, None], torch.arange(nkv, device=slot.device)
    at = (row, head, slot[..., None])  # [batch][ntok][nkv]
    out = {}
    x = st["qkv"].view(b, t, nq + 2 * nkv, hd)
    for n, heads in (("k", x[:, :, nq:nq + nkv]), ("v", x[:, :, nq + nkv:])):
        r = _rotate(heads)
        codes, scales = _quant8(r) if case["bits"] == 8 else _quant4(r)
        st[n + "q"][at] = codes.to(st[n + "q"].dtype)
        st[n + "s"][at] = scales
        y = _unrotate(_values(st[n + "q"][at], st[n + "s"][at], case["bits"]))
        out[n] = torch.where(here[..., None, None], y, torch.zeros_like(y)).view(b * t, nkv * hd)
    return out


def _scores(q, qs, k, bits, dtype=F32):
    """q [..., m, hd] int8 codes against a cache (codes, scales) [..., n]: [..., m, n]."""
    if bits == 8:  # whole products below 2^24: the sums are exact
        return (q @ k[0].to(dtype).transpose(-1, -2)) * k[1].to(dtype)[..., None, :] * qs[..., None]
    return (q @ _values(*k, bits, dtype).flatten(-2).transpose(-1, -2)) * qs[..., None]


def _plain_attn(case, st):
    n, beams, nq, nkv, hd = (case[x] for x in ("n_seq", "beams", "nq", "nkv", "hd"))
    g, bits, dev = nq // nkv, case["bits"], st["q"].device
    q, qs = _quant8(_rotate(st["q"].view(n, beams, nkv, g, hd)))
    qs = qs * (hd ** -0.5)
    # prefix: the group's rows [n][nkv][beams * g]; tails: [n * beams][nkv][g]
    by_head = lambda x: x.transpose(1, 2).flatten(2, 3)  # noqa: E731
    zp = _scores(by_head(q), by_head(qs), st["pk"], bits)
    zp = zp.masked_fill(torch.arange(zp.shape[-1], device=dev) >= st["plen"][:, None, None, None], -math.inf)
    zp = zp.unflatten(2, (beams, g)).transpose(1, 2)  # [n][beams][nkv][g][prefix]
    zt = _scores(q.flatten(0, 1), qs.flatten(0, 1), st["tk"], bits)
    zt = zt.masked_fill(torch.arange(zt.shape[-1], device=dev) >= st["tlen"][:, None, None, None], -math.inf)
    zt = zt.unflatten(0, (n, beams))
    m = torch.maximum(zp.amax(-1, keepdim=True), zt.amax(-1, keepdim=True))
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    pp, pt = torch.exp(zp - m), torch.exp(zt - m)
    total = (pp.sum(-1) + pt.sum(-1))[..., None]
    op = by_head(pp) @ _values(*st["pv"], bits).flatten(-2)
    ot = pt.flatten(0, 1) @ _values(*st["tv"], bits).flatten(-2)
    o = op.unflatten(2, (beams, g)).transpose(1, 2) + ot.unflatten(0, (n, beams))
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return _unrotate(o.unflatten(-1, (-1, 64))).reshape(n * beams, nq * hd)


def _plain_select(case, st):
    n, beams, v, k, eos = case["n_seq"], case["beams"], case["vocab"], case["k"], st["eos"]
    x = st["logits"].to(F64)
    x = torch.where(x.isnan(), torch.full_like(x, -math.inf), x).clamp(max=FLT_MAX)
    m = x.amax(-1, keepdim=True)
    z = x - torch.where(m == -math.inf, torch.zeros_like(m), m)
    score = st["scores"].to(F64)[:, None]
    s = score + (z - torch.log(torch.exp(z).sum(-1, keepdim=True)))
    token = torch.arange(v, device=x.device)
    ended = torch.where(token == eos, score, torch.full_like(score, -math.inf))
    s = torch.where(st["done"][:, None] != 0, ended, s)
    s = torch.where(s.isnan(), torch.full_like(s, -math.inf), s).view(n, beams * v)
    best, at = torch.sort(s, dim=-1, descending=True, stable=True)  # equal scores: the lowest index first
    best, at = best[:, :k], at[:, :k]
    none = best == -math.inf
    base = torch.arange(n, device=x.device)[:, None] * beams
    row, tok = torch.where(none, base, base + at // v), torch.where(none, torch.full_like(at, eos), at % v)
    done = none | (st["done"][row] != 0) | (tok == eos)
    return dict(scores=best.to(F32), tokens=tok.int(), parents=row.int(), done=done.int())


def _plain_reorder(case, st):
    to = st["parents"].long()
    here = torch.arange(case["cap"], device=to.device) < st["len"][to][:, None, None]  # [row][1][cap]
    for codes, scales in (st["k"], st["v"]):
        codes.copy_(torch.where(here[..., None], codes[:, to], codes))
        keep = here if case["bits"] == 8 else here[..., None]
        scales.copy_(torch.where(keep, scales[:, to], scales))
    return _flat(st)


# ---------------------------------------------------------------- the same in 64 bits
def _hadamard():
    i = np.arange(64)
    return 1.0 - 2.0 * (np.array([bin(a).count("1") for a in range(64)])[i[:, None] & i[None, :]] & 1)


def _codes(x, bits):
    """Codes (as the values they stand for, before their scale) and scales of heads x [..., hd]
    (numpy fp32): the format's own fp32 arithmetic, which codes next to a border depend on."""
    f = np.float32
    v = x.reshape(x.shape[:-1] + (-1, 64)) * np.array([_signs(b) for b in range(x.shape[-1] // 64)], f) * f(0.125)
    for h in (1, 2, 4, 8, 16, 32):
        low = (np.arange(64) & h) == 0
        a, b = v[..., low], v[..., ~low]
        v = np.empty_like(v)
        v[..., low], v[..., ~low] = a + b, a - b
    if bits == 8:
        mx = np.abs(v).max((-2, -1), keepdims=True)
        with np.errstate(divide="ignore", invalid="ignore"):
            q = np.where(mx <= FLT_EPS, f(0), np.rint(v * (f(127.0) / mx)))
        return q, np.where(mx <= FLT_EPS, f(0), mx / f(127.0))
    mid, cb = np.array(NF4_MID, f), np.array(NF4_CB, f)

    def nearest(y):
        p = np.searchsorted(mid, np.abs(y), side="right")
        return np.where(y >= 0, 8 + p, 7 - p)

    mx = np.abs(v).max(-1, keepdims=True)
    c = cb[nearest(v * (f(127.0) / mx))]
    num = np.add.accumulate(v * c, axis=-1, dtype=f)[..., -1:]
    den = (c * c).sum(-1, keepdims=True)
    s = torch.from_numpy(np.where(num > 0, num / den, mx / f(127.0))).to(torch.bfloat16).float().numpy()
    return cb[nearest(v * (f(1.0) / s))], s


def _unrot64(v):
    """Inverse rotation of [..., blocks, 64] in 64 bits, on the GPU."""
    h = torch.from_numpy(_hadamard()).to(v.device) / 8.0
    return ((v @ h) * _sign_rows(v.shape[-2], F64, str(v.device))).flatten(-2)


def exact(case, seed):
    if case["kind"] == "kv":
        qkv, _, count = _kv_inputs(case, seed)
        b, t, nq, nkv, hd = (case[x] for x in ("batch", "ntok", "nq", "nkv", "hd"))
        x = qkv.cpu().numpy().reshape(b, t, nq + 2 * nkv, hd)
        gone = torch.arange(t, device=DEV) >= count[:, None]
        out = {}
        for n, heads in (("k", x[:, :, nq:nq + nkv]), ("v", x[:, :, nq + nkv:])):
            q, s = _codes(heads, case["bits"])
            y = _unrot64(torch.from_numpy(q.astype(np.float64) * s).to(DEV))
            y[gone] = 0.0
            out[n] = y.reshape(b * t, nkv * hd)
        return out
    if case["kind"] == "attn":
        q, pk, pv, tk, tv, plen, tlen = _attn_inputs(case, seed)
        n, beams, nq, nkv, hd = (case[x] for x in ("n_seq", "beams", "nq", "nkv", "hd"))
        g, bits = nq // nkv, case["bits"]
        code, qs = _codes(q.cpu().numpy().reshape(n, beams, nkv, g, hd), 8)
        qv = torch.from_numpy(code.astype(np.float64) * qs).flatten(-2).to(DEV) / math.sqrt(hd)
        out = torch.zeros(n, beams, nkv, g, hd, dtype=F64, device=DEV)
        for s in range(n):
            for h in range(nkv):
                a = int(plen[s])
                k0, v0 = (_values(c[s, h, :a], w[s, h, :a], bits, F64).flatten(-2) for c, w in (pk, pv))
                z0 = qv[s, :, h] @ k0.T  # [beams][g][prefix]
                for r in range(beams):
                    row, e = s * beams + r, int(tlen[s * beams + r])
                    k1, v1 = (_values(c[row, h, :e], w[row, h, :e], bits, F64).flatten(-2) for c, w in (tk, tv))
                    p = torch.softmax(torch.cat((z0[r], qv[s, r, h] @ k1.T), -1), -1)
                    out[s, r, h] = p[:, :a] @ v0 + p[:, a:] @ v1
        return _unrot64(out.unflatten(-1, (-1, 64))).reshape(n * beams, nq * hd)
    if case["kind"] == "select":
        logits, scores, done = _select_inputs(case, seed)
        n, beams, k = case["n_seq"], case["beams"], case["k"]
        every = scores.to(F64)[:, None] + torch.log_softmax(logits.to(F64), -1)
        every[done != 0] = -math.inf
        every[done != 0, 2] = scores.to(F64)[done != 0]
        return dict(scores=every.view(n, -1).topk(k, -1).values, tokens=None, parents=None, done=None)
    k, v, parents = _reorder_inputs(case, seed)
    out = {}
    for name, (_, scales) in (("k", k), ("v", v)):
        new = scales.to(F64)
        for row, src in enumerate(parents.tolist()):
            new[:, row, :, :case["len"]] = scales[:, src, :, :case["len"]].to(F64)
        out[name + "s"] = new
    return dict(kq=None, ks=out["ks"], vq=None, vs=out["vs"])
