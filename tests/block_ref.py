"""The operators for blocks of tokens in plain numpy, 64 bits (query codes come from the oracle's
quantizer, whose fp32 arithmetic the cache format fixes)."""
import numpy as np

import branch_ref as B
import oracle as O

U = B.U  # half a step of fp32


def turns(rot, theta, scaling="plain", factor=1.0, original=0, low=0.0, high=0.0):
    """(turns per position of every pair as long doubles, factor of rotated elements)."""
    ld = np.longdouble
    i = np.arange(rot // 2, dtype=ld)
    two_pi = 2 * ld(np.pi) + ld(2.4492935982947064e-16)
    if scaling == "base":
        theta = ld(theta) * ld(factor) ** (ld(rot) / (rot - 2))
    f = ld(theta) ** (-2 * i / rot)
    keep, scale = np.ones_like(f), 1.0
    if scaling == "linear":
        keep[:] = 0
    elif scaling == "ramp":
        pair = lambda t: rot * np.log(original / (t * 2 * np.pi)) / (2 * np.log(float(theta)))  # noqa: E731
        a, b = max(np.floor(pair(high or 32.0)), 0.0), min(np.ceil(pair(low or 1.0)), rot - 1.0)
        keep = 1 - np.clip((i - a) / max(b - a, 0.001), 0, 1)
        scale = 0.1 * np.log(factor) + 1.0
    elif scaling == "wave":
        keep = np.clip((original * f / two_pi - (low or 1.0)) / ((high or 4.0) - (low or 1.0)), 0, 1)
    return (f * keep + f / ld(factor) * (1 - keep)) / two_pi, scale


def rope(x, pos, turn, scale, interleaved):
    """Heads x [tokens][heads][hd] at positions pos [tokens]: (out, bound). Cosine and sine are rounded once
    and their angles off by p * 2^-52 turns (the plan's rounding and the product's); two products and a sum
    round once each: four roundings of |x0 c| + |x1 s|."""
    n = len(turn)
    t = pos.astype(np.longdouble)[:, None] * turn
    a = ((t - np.rint(t)) * 2 * np.pi).astype(np.float64)[:, None]
    c, s = np.cos(a) * scale, np.sin(a) * scale
    lo, hi = (2 * np.arange(n), 2 * np.arange(n) + 1) if interleaved else (np.arange(n), np.arange(n) + n)
    out, bound = x.astype(np.float64), np.zeros(x.shape)
    x0, x1 = out[..., lo].copy(), out[..., hi].copy()
    off = 2 * np.pi * (np.abs(t) * 2.0 ** -52).astype(np.float64)[:, None] * scale
    out[..., lo], out[..., hi] = x0 * c - x1 * s, x1 * c + x0 * s
    bound[..., lo] = 4 * U * (np.abs(x0 * c) + np.abs(x1 * s)) + off * (np.abs(x0) + np.abs(x1))
    bound[..., hi] = 4 * U * (np.abs(x1 * c) + np.abs(x0 * s)) + off * (np.abs(x0) + np.abs(x1))
    return out, bound + 1e-44


def visible(ntok, start, count, length, sees=None):
    """bool [ntok][length]: what each token of a row sees of positions 0 .. length - 1."""
    p = np.arange(length)[None] - start
    t = np.arange(ntok)[:, None]
    inside = (p >= 0) & (p < count)
    if sees is None:
        return (p < 0) | (inside & (p <= t))
    bit = np.array([[sees[i] >> int(j) & 1 if 0 <= j < 64 else 0 for j in p[0]] for i in range(ntok)], bool)
    return (p < 0) | (inside & bit)


def attention(bits, q, cache, pos, counts, sees, nq, nkv, hd, scale, length):
    """q [batch][ntok][nq][hd]: (out, bound), NaN where a token is not there.

    With S the largest score (NF4: sum of its blocks' parts): a score is off by 4 roundings (dots are exact; 5 with two
    blocks), the exponent's argument by 2 more of a number up to 2 S, exp by 4, so a weight by (9 S + 4) u
    relative to its sum, twice (weights and their total). Terms are added 32 at a time, one group after the other,
    and in up to 64 parts: n / 32 + 128 roundings; a weight held in two 11-bit pieces by 2^-21. All relative to the
    sum of absolute terms; the inverse rotation adds a block's 64 errors over 8 and 7 roundings of its own."""
    batch, ntok = q.shape[:2]
    out, bound = np.full((batch, ntok, nq, hd), np.nan), np.full((batch, ntok, nq, hd), np.nan)
    for r in range(batch):
        count = int(max(0, min(ntok, counts[r])))
        see = visible(ntok, int(pos[r]), count, length, None if sees is None else [int(x) for x in sees[r]])
        for h in range(nkv):
            with np.errstate(invalid="ignore", over="ignore"):
                k, v = (B.values(bits, cache[i][r, h, :length], cache[i + 1][r, h, :length]) for i in (0, 2))
            for t in range(count):
                at = np.nonzero(see[t])[0]
                n = len(at)
                for g in range(nq // nkv):
                    head = h * (nq // nkv) + g
                    if n == 0:
                        out[r, t, head] = bound[r, t, head] = 0.0
                        continue
                    code, qs = O.kv_quant_head(q[r, t, head])
                    qv = code.astype(np.float64) * np.float64(qs) * float(np.float32(scale))
                    parts = (k[at] * qv).reshape(n, hd // 64, 64).sum(-1) if bits == 4 else (k[at] @ qv)[:, None]
                    z, S = parts.sum(-1), np.abs(parts).sum(-1).max()
                    p = np.exp(z - z.max())
                    p /= p.sum()
                    o, size = p @ v[at], p @ np.abs(v[at])
                    rel = (2 * (9 * S + 4) + 2 * (n / 32 + 128)) * U + 2.0 ** -21
                    out[r, t, head] = B.unrotate(o)
                    bound[r, t, head] = (rel * B.block_sums(size) + 7 * U * B.block_sums(np.abs(o))) / 8 + 1e-37
    return out, bound


def logits(x, vocab, rules):
    """Rows of logits after the rules (a dict of host arrays), rounded once."""
    out = x.copy()
    R = rules.get
    for r in range(x.shape[0]):
        y = {}
        if R("history") is not None:
            h = R("history")[r]
            if R("history_len") is not None:
                h = h[:max(0, R("history_len")[r])]
            prompt = 0 if R("prompt_len") is None else R("prompt_len")[r]
            inside = lambda a: a[(a >= 0) & (a < vocab)]  # noqa: E731
            count = np.bincount(inside(h[max(0, prompt):]), minlength=vocab)
            for t in np.unique(inside(h)):
                v = np.float64(x[r, t])
                rep = np.float64(1.0 if R("repeat") is None else R("repeat")[r])
                v = v / rep if v > 0 else v * rep
                if count[t]:
                    v = v - (np.float64(0.0 if R("presence") is None else R("presence")[r]) +
                             np.float64(0.0 if R("frequency") is None else R("frequency")[r]) * np.float64(count[t]))
                y[int(t)] = v
        if R("bias") is not None:
            n = R("bias").shape[1] if R("bias_len") is None else min(R("bias").shape[1], max(0, R("bias_len")[r]))
            for t, b in zip(R("bias_tokens")[r, :n], R("bias")[r, :n]):
                if 0 <= t < vocab:
                    y[int(t)] = y.get(int(t), np.float64(x[r, t])) + np.float64(b)
        for t, v in y.items():
            out[r, t] = np.float32(v)
        if R("mask") is not None:
            m = r if R("mask_row") is None else R("mask_row")[r]
            if 0 <= m < R("mask").shape[0]:
                bit = np.unpackbits(np.ascontiguousarray(R("mask")[m]).view(np.uint8), bitorder="little")[:vocab]
                out[r, :vocab][bit == 0] = -np.inf
    return out


def keep(arrays, pos, keep_, counts, n_keep):
    """Each array [layers][rows][nkv][cap][...] with its rows' kept positions moved."""
    out = [a.copy() for a in arrays]
    cap = arrays[0].shape[3]
    for r in range(arrays[0].shape[1]):
        n = n_keep if counts is None else max(0, min(n_keep, int(counts[r])))
        for j in range(n):
            src, to = int(pos[r]) + int(keep_[r, j]), int(pos[r]) + j
            if keep_[r, j] >= j and 0 <= to and src < cap:
                for a, o in zip(arrays, out):
                    o[:, r, :, to] = a[:, r, :, src]
    return out
