"""The operators for several continuations of one prompt in plain numpy, 64 bits (codes come from
the oracle's quantizers, whose fp32 arithmetic the cache format fixes)."""
import numpy as np

import oracle as O

NF4 = np.array([-127, -96, -75, -58, -44, -31, -18, -6, 6, 18, 31, 44, 58, 75, 96, 127], np.float64)
U = 2.0 ** -24  # half a step of fp32


def new_cache(bits, rows, nkv, cap, hd, rng=None):
    """(kq, ks, vq, vs) of rows x nkv x cap slots: a byte pattern, or random codes and scales."""
    shape = (rows, nkv, cap)
    out = []
    for _ in range(2):
        if bits == 8:
            q = np.full(shape + (hd,), 0x5A, np.int8) if rng is None else rng.integers(-127, 128, shape + (hd,)).astype(np.int8)
            s = np.full(shape, 7.5, np.float32) if rng is None else rng.uniform(0.005, 0.05, shape).astype(np.float32)
        else:
            q = np.full(shape + (hd // 2,), 0x5A, np.uint8) if rng is None else rng.integers(0, 256, shape + (hd // 2,)).astype(np.uint8)
            f = np.full(shape + (hd // 64,), 7.5, np.float32) if rng is None else \
                rng.uniform(0.005, 0.05, shape + (hd // 64,)).astype(np.float32)
            s = (f.view(np.uint32) >> 16).astype(np.uint16)
        out += [q, s]
    return out


def store(bits, head):
    return O.kv_quant_head(head) if bits == 8 else O.kv_quant_head_q4(head)


def bf16(s):
    return (s.astype(np.uint32) << 16).view(np.float32)


def values(bits, q, s):
    """Rotated heads [..., hd] that codes and scales stand for, 64 bits."""
    if bits == 8:
        with np.errstate(invalid="ignore"):  # (slots that hold nothing may carry any scale)
            return q.astype(np.float64) * s.astype(np.float64)[..., None]
    b = q.reshape(q.shape[:-1] + (-1, 2, 16))
    v = NF4[np.stack((b & 15, b >> 4), -2)].reshape(q.shape[:-1] + (-1, 64))
    return (v * bf16(s).astype(np.float64)[..., None]).reshape(q.shape[:-1] + (-1,))


def unrotate(v):
    """ifwht64 of every 64-block, 64 bits."""
    i = np.arange(64)
    h = 1.0 - 2.0 * (np.array([bin(a).count("1") for a in range(64)])[i[:, None] & i[None, :]] & 1)
    b = v.reshape(v.shape[:-1] + (-1, 64))
    sign = np.array([[1.0 - 2.0 * (O.sign_bits(k) >> j & 1) for j in range(64)] for k in range(b.shape[-2])])
    return ((b @ h) * sign / 8.0).reshape(v.shape)


def block_sums(a):
    """Sum of every 64-block, spread over it."""
    b = a.reshape(a.shape[:-1] + (-1, 64))
    return np.broadcast_to(b.sum(-1, keepdims=True), b.shape).reshape(a.shape)


def attention(bits, q, prefix, tail, plen, tlen, beams, nq, nkv, hd, scale):
    """(out, bound) [rows][nq][hd]; bound: how far fp32 arithmetic may be off, element by element.

    With S the largest score: a score is off by 4 roundings (the dot is exact), the exponent's
    argument by 2 more of a number up to 2 S, exp by 4, so a weight by (4 S + 4 S + 4) u relative
    to its sum, twice (weights and their total).  A sum of n terms in workgroups of 256 positions
    and n / 256 parts is off by 256 + n / 256 + 32 roundings; a weight held in two 11-bit pieces by
    2^-21.  All relative to the sum of absolute terms; the inverse rotation adds a block's 64
    errors over 8 and 7 roundings of its own."""
    rows = q.shape[0]
    out = np.zeros((rows, nq, hd))
    bound = np.zeros((rows, nq, hd))
    pk, pv, tk, tv = (values(bits, *c) for c in (prefix[:2], prefix[2:], tail[:2], tail[2:]))
    for r in range(rows):
        s, a, e = r // beams, int(plen[r // beams]), int(tlen[r])
        for h in range(nq):
            g = h // (nq // nkv)
            code, qs = O.kv_quant_head(q[r, h])
            k = np.concatenate((pk[s, g, :a], tk[r, g, :e]))
            v = np.concatenate((pv[s, g, :a], tv[r, g, :e]))
            n = len(k)
            if n == 0:
                continue
            z = (k @ (code.astype(np.float64) * np.float64(qs))) * float(np.float32(scale))
            p = np.exp(z - z.max())
            p /= p.sum()
            o, size = p @ v, p @ np.abs(v)
            rel = (2 * (8 * np.abs(z).max() + 4) + 2 * (288 + n / 256)) * U + 2.0 ** -21
            out[r, h] = unrotate(o)
            bound[r, h] = (rel * block_sums(size) + 7 * U * block_sums(np.abs(o))) / 8 + 1e-37
    return out, bound


def select(logits, scores, done, n_seq, beams, k, eos):
    """(scores64, tokens, parents, done) [n_seq][k], and the smallest gap between neighbours of
    different rows in the order, up to the first candidate left out."""
    v = logits.shape[1]
    x = np.where(np.isnan(logits), -np.inf, np.minimum(logits, np.finfo(np.float32).max)).astype(np.float64)
    out = [], [], [], []
    gap = np.inf
    for s in range(n_seq):
        cand = []
        for b in range(beams):
            r = s * beams + b
            sc = np.float64(scores[r])
            if not sc > -np.inf:
                continue
            if done is not None and done[r]:
                cand.append((-sc, b, 0.0, eos))
                continue
            live = np.nonzero(x[r] > -np.inf)[0]
            if not len(live):
                continue
            m = x[r].max()
            lp = (x[r, live] - m) - np.log(np.exp(x[r, live] - m).sum())
            best = live[np.lexsort((live, -x[r, live]))][:k]
            pos = {t: i for i, t in enumerate(live)}
            cand += [(-(sc + lp[pos[t]]), b, -x[r, t], int(t)) for t in best]
        cand.sort()
        for a, c in zip(cand[:k], cand[1:k + 1]):
            if a[1] != c[1] and a[0] != c[0]:
                gap = min(gap, c[0] - a[0])
        picks = cand[:k]
        fill = k - len(picks)
        out[0].append([-p[0] for p in picks] + [-np.inf] * fill)
        out[1].append([p[3] for p in picks] + [max(eos, 0)] * fill)
        out[2].append([s * beams + p[1] for p in picks] + [s * beams] * fill)
        out[3].append([int(bool(done is not None and done[s * beams + p[1]]) or p[3] == eos) for p in picks] + [1] * fill)
    return tuple(np.array(o) for o in out) + (gap,)
