"""Several continuations of one prompt: the batched Hadamard cache (k2t_kv_append, k2t_kv_load,
k2t_kv_reorder), attention over a shared prefix (k2t_attn_shared) and beam search's choice
(k2t_beam_select), against 64-bit references (branch_ref) and the one-sequence operators."""

import numpy as np
import pytest
import torch

import branch_ref as R
import k2t

pytestmark = pytest.mark.gpu


def dev(a):
    a = np.ascontiguousarray(a)
    return torch.from_numpy(a.view(np.int16) if a.dtype == np.uint16 else a).cuda()


def host(t, like):
    return t.cpu().numpy().view(like.dtype)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def rows_of(cache, cap, length=None, d_len=None):
    t = [dev(a) for a in cache]
    return t, k2t.KVRows(*t, cap=cap, len=length, d_len=d_len)


def workspace(n):
    return torch.full((n,), 0x7F, dtype=torch.uint8, device="cuda")


# ---------------------------------------------------------------- append, load
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("batch,ntok,nkv,cap", [(1, 1, 1, 1), (3, 5, 2, 9), (2, 70, 3, 71), (5, 1, 4, 3)])
def test_append_writes_kv_stores_bytes_and_load_reads_them(gpu_ctx, bits, hd, batch, ntok, nkv, cap):
    print(f"kv_append bits={bits} hd={hd} batch={batch} ntok={ntok} nkv={nkv} cap={cap}", flush=True)
    rng = np.random.default_rng(bits * hd + ntok)
    width = 2 * nkv * hd + hd + 4  # a q head in front, padding behind
    x = (rng.standard_normal((batch * ntok, width)) * rng.uniform(0.01, 4, (batch * ntok, 1))).astype(np.float32)
    x[0, hd:2 * hd] = 0.0  # a zero head
    pos = rng.integers(-2, cap + 1, batch).astype(np.int32)
    counts = rng.integers(0, ntok + 2, batch).astype(np.int32)
    pos[0], counts[0] = 0, ntok
    want = R.new_cache(bits, batch, nkv, cap, hd)
    (kq, ks, vq, vs), kv = rows_of(want, cap)
    dx = dev(x)
    at = dx.data_ptr() + 4 * hd
    gpu_ctx.kv_append(bits, at, at + 4 * nkv * hd, width, batch, ntok, nkv, hd, dev(pos), kv, counts=dev(counts))
    got_k = torch.full((batch * ntok, nkv * hd + 8), 3.25, device="cuda")
    got_v = got_k.clone()
    gpu_ctx.kv_load(bits, kv, batch, ntok, nkv, hd, dev(pos), got_k, got_v, nkv * hd + 8, counts=dev(counts))
    gpu_ctx.sync()
    load = [np.full((batch * ntok, nkv * hd + 8), 3.25) for _ in range(2)]
    tol = [np.zeros_like(a) for a in load]
    for b in range(batch):
        for t in range(min(ntok, counts[b])):
            p = pos[b] + t
            if not 0 <= p < cap:
                continue
            for h in range(nkv):
                for w in range(2):
                    o = hd + (w * nkv + h) * hd
                    q, s = R.store(bits, x[b * ntok + t, o:o + hd])
                    want[2 * w][b, h, p], want[2 * w + 1][b, h, p] = q, s
                    v = R.values(bits, want[2 * w][b, h, p], want[2 * w + 1][b, h, p])
                    load[w][b * ntok + t, h * hd:(h + 1) * hd] = R.unrotate(v)
                    # code * scale, then six sums and a division by 8: 7 roundings of a block's sum
                    tol[w][b * ntok + t, h * hd:(h + 1) * hd] = 7.5 * R.U * R.block_sums(np.abs(v)) / 8
    for g, w in zip((kq, ks, vq, vs), want):
        assert np.array_equal(host(g, w).view(np.uint8), w.view(np.uint8))
    for g, w, t in zip((got_k, got_v), load, tol):
        assert (np.abs(g.cpu().numpy() - w) <= t).all()


@pytest.mark.parametrize("bits", [8, 4])
def test_append_equals_kv_store(gpu_ctx, bits):
    rng = np.random.default_rng(5)
    hd, n = 128, 33
    x = dev(rng.standard_normal((n, 2 * hd)).astype(np.float32))
    a, kv = rows_of(R.new_cache(bits, 1, 1, n, hd), n)
    gpu_ctx.kv_append(bits, x, x.data_ptr() + 4 * hd, 2 * hd, 1, n, 1, hd, ints([0]), kv)
    b, _ = rows_of(R.new_cache(bits, 1, 1, n, hd), n)
    gpu_ctx.kv_store(bits, x[:, :hd].contiguous(), n, hd, b[0], b[1])
    gpu_ctx.kv_store(bits, x[:, hd:].contiguous(), n, hd, b[2], b[3])
    gpu_ctx.sync()
    assert all(torch.equal(u, v) for u, v in zip(a, b))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd", [64, 128])
def test_append_of_odd_values_equals_kv_store(gpu_ctx, bits, hd):
    """Heads that hold NaN, infinities, the largest and smallest floats, one value, or nothing but -0."""
    rng = np.random.default_rng(hd)
    kinds = [np.nan, -np.nan, np.inf, -np.inf, 3e38, -3e38, 1e-38, 1e-45, -0.0, 1e-31, 1.2e-7, 1.0]
    x = []
    for v in kinds:
        a, b, c = rng.standard_normal(hd), np.full(hd, v), np.zeros(hd)
        a[rng.integers(hd)] = v
        c[hd - 1] = v
        x += [a, b, c, np.where(np.arange(hd) < 32, v, -v)]
    x = np.array(x, np.float32)
    n = len(x)
    dx = dev(x)
    a, kv = rows_of(R.new_cache(bits, 1, 1, n, hd), n)
    gpu_ctx.kv_append(bits, dx, dx, hd, 1, n, 1, hd, ints([0]), kv)
    b, _ = rows_of(R.new_cache(bits, 1, 1, n, hd), n)
    gpu_ctx.kv_store(bits, dx, n, hd, b[0], b[1])
    gpu_ctx.sync()
    for i in range(2):
        assert np.array_equal(a[i].cpu().numpy().view(np.uint8), b[i].cpu().numpy().view(np.uint8))
        assert np.array_equal(a[i + 2].cpu().numpy().view(np.uint8), b[i].cpu().numpy().view(np.uint8))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd", [64, 128])
def test_append_and_load_of_many_tokens(gpu_ctx, bits, hd):
    """Enough blocks for two per group of lanes, ragged rows: append against k2t_kv_store's bytes, load
    against append's."""
    g = torch.Generator(device="cuda").manual_seed(hd + bits)
    batch, ntok, nkv = 3, 701, 2048 // hd
    x = torch.randn(batch * ntok, 2 * nkv * hd, generator=g, device="cuda")
    counts, pos, cap = [701, 350, 699], [0, 3, 2], 704
    want, _ = rows_of(R.new_cache(bits, batch, nkv, cap, hd), cap)
    a, kv = rows_of(R.new_cache(bits, batch, nkv, cap, hd), cap)
    q, s = (torch.empty((batch * ntok * nkv,) + t.shape[3:], dtype=t.dtype, device="cuda") for t in want[:2])
    for w in range(2):
        heads = x[:, w * nkv * hd:(w + 1) * nkv * hd].contiguous()
        gpu_ctx.kv_store(bits, heads, batch * ntok * nkv, hd, q, s)
        gpu_ctx.sync()
        for b in range(batch):
            for got, t in ((q, want[2 * w]), (s, want[2 * w + 1])):
                rows = got.view((batch, ntok, nkv) + t.shape[3:])[b, :counts[b]].transpose(0, 1)
                t[b, :, pos[b]:pos[b] + counts[b]] = rows
    at = x.data_ptr()
    gpu_ctx.kv_append(bits, at, at + 4 * nkv * hd, 2 * nkv * hd, batch, ntok, nkv, hd, ints(pos), kv, counts=ints(counts))
    y = torch.full_like(x, 9.0)
    gpu_ctx.kv_load(bits, kv, batch, ntok, nkv, hd, ints(pos), y.data_ptr(), y.data_ptr() + 4 * nkv * hd, 2 * nkv * hd,
                    counts=ints(counts))
    gpu_ctx.sync()
    assert all(torch.equal(u, v) for u, v in zip(a, want))
    for b in range(batch):
        rows = y.view(batch, ntok, 2, nkv, hd)[b]
        assert bool((rows[counts[b]:] == 9.0).all())
        for w in range(2):
            n = counts[b]
            vals = R.values(bits, host(a[2 * w][b, :, pos[b]:pos[b] + n], np.zeros(0, np.int8 if bits == 8 else np.uint8)),
                            host(a[2 * w + 1][b, :, pos[b]:pos[b] + n], np.zeros(0, np.float32 if bits == 8 else np.uint16)))
            err = np.abs(rows[:n, w].cpu().numpy().transpose(1, 0, 2) - R.unrotate(vals))
            assert (err <= 7.5 * R.U * R.block_sums(np.abs(vals)) / 8).all()


def test_append_offsets_past_32_bits(gpu_ctx):
    """A cache of 2^20 positions x 40 heads of 128 bytes (5 GiB): the last head's last slot."""
    hd, nkv, cap = 128, 40, 1 << 20
    q = torch.zeros(nkv * cap, hd, dtype=torch.int8, device="cuda")
    s = torch.zeros(nkv * cap, device="cuda")
    kv = k2t.KVRows(q, s, q, s, cap=cap)  # (K and V alike, so one buffer serves for both)
    x = torch.randn(1, nkv * hd, device="cuda")
    gpu_ctx.kv_append(8, x, x, nkv * hd, 1, 1, nkv, hd, ints([cap - 1]), kv)
    y = torch.zeros_like(x)
    gpu_ctx.kv_load(8, kv, 1, 1, nkv, hd, ints([cap - 1]), y, torch.zeros_like(x), nkv * hd)
    gpu_ctx.sync()
    rq, rs = R.store(8, x[0, -hd:].cpu().numpy())
    assert np.array_equal(q[-1].cpu().numpy(), rq) and float(s[-1]) == float(rs)
    # half a code step of each head's scale, per rotated element: 8 in all after the rotation
    assert float((x - y).abs().max()) <= 64 / 8 * 0.51 * float(s.max())
    assert int((q != 0).any(1).sum()) == nkv


# ---------------------------------------------------------------- reorder
@pytest.mark.parametrize("bits,hd", [(8, 64), (8, 128), (4, 64), (4, 128)])
@pytest.mark.parametrize("layers,n_seq,beams,nkv,cap,length", [(1, 1, 2, 1, 5, 5), (2, 3, 4, 2, 33, 30), (1, 2, 13, 3, 70, 1),
                                                               (3, 1, 31, 1, 20, 19), (1, 1, 64, 2, 300, 290)])
def test_reorder_moves_rows_in_place(gpu_ctx, bits, hd, layers, n_seq, beams, nkv, cap, length):
    print(f"kv_reorder bits={bits} hd={hd} {layers} {n_seq} {beams} {nkv} {cap} {length}", flush=True)
    rng = np.random.default_rng(beams + hd)
    rows = n_seq * beams
    cache = R.new_cache(bits, layers * rows, nkv, cap, hd, rng)
    lens = rng.integers(0, length + 1, rows).astype(np.int32)
    lens[rng.integers(rows)] = length
    parents = np.concatenate([s * beams + rng.integers(0, beams, beams) for s in range(n_seq)]).astype(np.int32)
    parents[0] = rows if rows < 2 else -5  # a parent outside its sequence
    if n_seq > 1:
        parents[-1] = 0  # another sequence's row
    want = []
    for a in cache:
        a = a.reshape((layers, rows) + a.shape[1:])
        new = a.copy()
        for r in range(rows):
            p = parents[r]
            if p // beams == r // beams and 0 <= p < rows:
                new[:, r, :, :lens[p]] = a[:, p, :, :lens[p]]
        want.append(new)
    t, kv = rows_of(cache, cap, length, dev(lens))
    gpu_ctx.kv_reorder(bits, kv, dev(parents), layers, n_seq, beams, nkv, hd)
    gpu_ctx.sync()
    for g, w in zip(t, want):
        assert np.array_equal(host(g, w).reshape(-1), w.reshape(-1))


# ---------------------------------------------------------------- attention
ATTN = [
    # n_seq, beams, nq, nkv, prefix, tail
    (1, 1, 1, 1, 1, 0), (1, 1, 4, 4, 0, 1), (1, 4, 9, 3, 45, 7), (2, 3, 8, 2, 63, 65), (1, 5, 4, 4, 257, 31),
    (1, 17, 8, 1, 130, 3), (3, 2, 24, 2, 513, 20), (1, 3, 2, 1, 9000, 5), (2, 40, 4, 4, 700, 2), (1, 2, 40, 2, 600, 150), (1, 33, 4, 2, 1000, 33), (1, 1, 16, 1, 700, 300), (1, 64, 2, 1, 31, 2),
]


@pytest.mark.parametrize("bits,hd", [(8, 64), (8, 128), (4, 64), (4, 128)])
@pytest.mark.parametrize("n_seq,beams,nq,nkv,prefix,tail", ATTN)
def test_attention_over_prefix_and_tail(gpu_ctx, bits, hd, n_seq, beams, nq, nkv, prefix, tail):
    print(f"attn_shared bits={bits} hd={hd} {n_seq} {beams} {nq} {nkv} {prefix} {tail}", flush=True)
    rng = np.random.default_rng(prefix + tail + hd + bits)
    rows, pcap, tcap = n_seq * beams, max(prefix, 1) + 3, max(tail, 1) + 2
    pre, tl = R.new_cache(bits, n_seq, nkv, pcap, hd, rng), R.new_cache(bits, rows, nkv, tcap, hd, rng)
    plen = rng.integers(prefix // 2, prefix + 1, n_seq).astype(np.int32)
    tlen = rng.integers(0, tail + 1, rows).astype(np.int32)
    plen[0], tlen[-1] = prefix, tail
    for c, n in ((pre, plen), (tl, tlen)):  # what lies behind a row's positions is never used
        for r in range(len(n)):
            if bits == 8:
                c[1][r, :, n[r]:] = np.nan
                c[3][r, :, n[r]:] = np.inf
            else:
                c[1][r, :, n[r]:] = 0x7FC0
                c[3][r, :, n[r]:] = 0x7F80
    width = nq * hd + 4
    q = (2 * rng.standard_normal((rows, width))).astype(np.float32)
    scale = hd ** -0.5
    out = torch.full((rows, nq, hd), float("nan"), device="cuda")
    _, p = rows_of(pre, pcap, prefix, dev(plen))
    _, t = rows_of(tl, tcap, tail, dev(tlen))
    ws = workspace(gpu_ctx.attn_shared_workspace(n_seq, beams, nq, nkv, hd, prefix, tail))
    gpu_ctx.attn_shared(bits, dev(q), width, n_seq, beams, nq, nkv, hd, p, t, scale, out, ws)
    gpu_ctx.sync()
    want, bound = R.attention(bits, q[:, :nq * hd].reshape(rows, nq, hd), pre, tl, plen, tlen, beams, nq, nkv, hd, scale)
    err = np.abs(out.cpu().numpy() - want)
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("bits,hd", [(8, 64), (8, 128), (4, 64), (4, 128)])
def test_attention_of_many_rows(gpu_ctx, bits, hd):
    """Enough rows and positions for the prefix items of two tiles of columns (18304 steps); the last
    item holds one tile."""
    rng = np.random.default_rng(hd + bits)
    beams, nq, nkv, prefix, tail = 61, 32, 8, 4600, 3
    pre, tl = R.new_cache(bits, 1, nkv, prefix, hd, rng), R.new_cache(bits, beams, nkv, tail, hd, rng)
    q = (2 * rng.standard_normal((beams, nq, hd))).astype(np.float32)
    out = torch.full((beams, nq, hd), float("nan"), device="cuda")
    _, p = rows_of(pre, prefix)
    _, t = rows_of(tl, tail)
    ws = workspace(gpu_ctx.attn_shared_workspace(1, beams, nq, nkv, hd, prefix, tail))
    gpu_ctx.attn_shared(bits, dev(q.reshape(beams, -1)), nq * hd, 1, beams, nq, nkv, hd, p, t, hd ** -0.5, out, ws)
    gpu_ctx.sync()
    rows = [0, 1, 30, 59, 60]  # (the reference of a few rows)
    want, bound = R.attention(bits, q[rows], pre, [a[rows] for a in tl], [prefix], [tail] * 5, 5, nq, nkv, hd, hd ** -0.5)
    err = np.abs(out.cpu().numpy()[rows] - want)
    assert (err <= bound).all(), float((err / bound).max())
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("bits,hd", [(8, 64), (8, 128), (4, 64), (4, 128)])
def test_attention_without_positions_prefix_or_tail(gpu_ctx, bits, hd):
    """Rows that hold nothing get zeros; a missing cache is one of no positions; lengths beyond
    `len` or below zero count as `len` and zero."""
    rng = np.random.default_rng(hd)
    beams, nq, nkv = 3, 4, 2
    pre, tl = R.new_cache(bits, 1, nkv, 40, hd, rng), R.new_cache(bits, beams, nkv, 9, hd, rng)
    q = rng.standard_normal((beams, nq * hd)).astype(np.float32)
    ws = workspace(gpu_ctx.attn_shared_workspace(1, beams, nq, nkv, hd, 40, 9))
    none = R.new_cache(bits, beams, nkv, 1, hd, rng)
    for p_len, t_len in (([0], [0, 4, -3]), ([99], [99, 2, 9]), (None, [1, 0, 5]), ([17], None)):
        _, p = rows_of(pre, 40, 40, ints(p_len) if p_len else None)
        _, t = rows_of(tl, 9, 8, ints(t_len) if t_len else None)
        out = torch.full((beams, nq, hd), float("nan"), device="cuda")
        gpu_ctx.attn_shared(bits, dev(q), nq * hd, 1, beams, nq, nkv, hd, p if p_len else None, t if t_len else None,
                            0.125, out, ws)
        gpu_ctx.sync()
        a = np.clip(p_len or [0], 0, 40)
        b = np.clip(t_len or [0, 0, 0], 0, 8)
        want, bound = R.attention(bits, q.reshape(beams, nq, hd), pre, tl if t_len else none, a, b, beams, nq, nkv, hd, 0.125)
        err = np.abs(out.cpu().numpy() - want)
        assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("bits,hd", [(8, 128), (4, 64)])
@pytest.mark.parametrize("prefix", [50, 1500])
def test_attention_of_bad_rows_stays_in_them(gpu_ctx, bits, hd, prefix):
    """NaN and infinities in one row's query, K scales and V scales: the other rows' bits do not change."""
    rng = np.random.default_rng(prefix)
    beams, nq, nkv, tail = 6, 8, 2, 20
    pre, tl = R.new_cache(bits, 1, nkv, prefix, hd, rng), R.new_cache(bits, beams, nkv, tail, hd, rng)
    q = rng.standard_normal((beams, nq * hd)).astype(np.float32)
    ws = workspace(gpu_ctx.attn_shared_workspace(1, beams, nq, nkv, hd, prefix, tail))

    def run():
        _, p = rows_of(pre, prefix)
        _, t = rows_of(tl, tail)
        out = torch.zeros((beams, nq, hd), device="cuda")
        gpu_ctx.attn_shared(bits, dev(q), nq * hd, 1, beams, nq, nkv, hd, p, t, hd ** -0.5, out, ws)
        gpu_ctx.sync()
        return out.cpu().numpy()

    good = run()
    assert np.isfinite(good).all()
    q[1, 5], q[2, hd + 3] = np.nan, np.inf
    tl[1][3, 0, 7] = np.nan if bits == 8 else 0x7FC0
    tl[3][4, 1, 2] = np.inf if bits == 8 else 0x7F80
    bad = run()
    assert np.array_equal(bad[[0, 5]], good[[0, 5]])
    for r, heads in ((1, [0]), (2, [1]), (3, [0, 1, 2, 3]), (4, [4, 5, 6, 7])):  # nor do the row's other heads
        rest = [h for h in range(nq) if h not in heads]
        assert np.array_equal(bad[r, rest], good[r, rest])
        assert r == 1 or not np.isfinite(bad[r, heads]).all()


@pytest.mark.parametrize("bits,hd", [(8, 64), (4, 128)])
@pytest.mark.parametrize("first,last", [(0, 8192), (0, 12000), (8192, 12000), (5000, 5001)])
def test_attention_of_nan_over_many_parts(gpu_ctx, bits, hd, first, last):
    """NaN scores on end, for as many positions as the joining of the parts takes at a time: they reach the
    output, whatever the other positions hold."""
    rng = np.random.default_rng(first + last)
    beams, nq, nkv, prefix, tail = 2, 9, 3, 12000, 4
    pre, tl = R.new_cache(bits, 1, nkv, prefix, hd, rng), R.new_cache(bits, beams, nkv, tail, hd, rng)
    pre[1][:, 1, first:last] = np.nan if bits == 8 else 0x7FC0  # (the middle KV head's: q heads 3 to 5)
    q = rng.standard_normal((beams, nq * hd)).astype(np.float32)
    out = torch.zeros((beams, nq, hd), device="cuda")
    _, p = rows_of(pre, prefix)
    _, t = rows_of(tl, tail)
    ws = workspace(gpu_ctx.attn_shared_workspace(1, beams, nq, nkv, hd, prefix, tail))
    gpu_ctx.attn_shared(bits, dev(q), nq * hd, 1, beams, nq, nkv, hd, p, t, hd ** -0.5, out, ws)
    gpu_ctx.sync()
    out = out.cpu().numpy()
    assert np.isnan(out[:, 3:6]).all()
    assert np.isfinite(out[:, :3]).all() and np.isfinite(out[:, 6:]).all()


@pytest.mark.parametrize("bits", [8, 4])
def test_attention_weights_far_apart_and_scales_of_any_size(gpu_ctx, bits):
    """One position takes all the weight, wherever it lies; V scales from 1e-12 to 1e12."""
    rng = np.random.default_rng(bits)
    beams, nq, nkv, hd, prefix, tail = 2, 2, 1, 64, 300, 40
    for spot in (0, 31, 32, 255, 256, 299, 300, 339):
        pre, tl = R.new_cache(bits, 1, nkv, prefix, hd, rng), R.new_cache(bits, beams, nkv, tail, hd, rng)
        size = np.float32(10.0 ** rng.uniform(-12, 12))
        for c in (pre, tl):
            if bits == 8:
                c[3][:] = c[3] * size
            else:
                c[3][:] = ((R.bf16(c[3]) * size).view(np.uint32) >> 16).astype(np.uint16)
        q = (30 * rng.standard_normal((beams, nq, hd))).astype(np.float32)
        for r in range(beams):
            c, row, pos = (pre, 0, spot) if spot < prefix else (tl, r, spot - prefix)
            if bits == 8:  # the position's K head is the query's own codes
                import oracle as O
                c[0][row, 0, pos], c[1][row, 0, pos] = O.kv_quant_head(q[r, 0])[0], 0.05
        out = torch.full((beams, nq, hd), float("nan"), device="cuda")
        _, p = rows_of(pre, prefix)
        _, t = rows_of(tl, tail)
        ws = workspace(gpu_ctx.attn_shared_workspace(1, beams, nq, nkv, hd, prefix, tail))
        gpu_ctx.attn_shared(bits, dev(q.reshape(beams, -1)), nq * hd, 1, beams, nq, nkv, hd, p, t, 0.125, out, ws)
        gpu_ctx.sync()
        want, bound = R.attention(bits, q, pre, tl, [prefix], [tail] * beams, beams, nq, nkv, hd, 0.125)
        err = np.abs(out.cpu().numpy() - want)
        assert (err <= bound).all(), (spot, float((err / bound).max()))


@pytest.mark.parametrize("bits,hd", [(8, 64), (8, 128), (4, 64), (4, 128)])
@pytest.mark.parametrize("beams,nq,nkv,prefix,tail", [(3, 4, 2, 50, 20), (3, 4, 2, 1500, 200), (61, 32, 8, 4600, 3)])
@pytest.mark.parametrize("kind", ["outlier", "spread", "sink", "blocks", "none"])
def test_attention_of_v_scales_far_apart(gpu_ctx, bits, hd, beams, nq, nkv, prefix, tail, kind):
    """V scales that differ from position to position (NF4: from block to block too). outlier: every tile
    of 32 holds a position of negligible weight whose scale is 2^30 times the others'; spread: any scales
    within 2^-30 .. 2^30; sink: the position that takes nearly all the weight holds a scale 2^-40 of the others',
    and every seventh V head is zero; blocks: the scales of NF4's second blocks are 2^-44 of the first's (2^44 in
    the tails); none: no V scale but zero in the first tiles.  Weights refer to products with V scales here, so an
    exponent is off by a rounding of up to 2 |z| / ln 2 + 44 + 17, which is 2 (|z| + 43) u in weight and total: within
    the bound's 2 (8 |z| + 4) u and the 2 x 43 u of its 2 x 288 that sums of at most 128 terms on end leave."""
    rng = np.random.default_rng(hd + bits + prefix)
    pre, tl = R.new_cache(bits, 1, nkv, prefix, hd, rng), R.new_cache(bits, beams, nkv, tail, hd, rng)
    for c in (pre, tl):
        n, rows = c[1].shape[2], c[1].shape[0]
        # all positions' K heads agree with the queries in element 0, those of `apart` oppose them
        apart = np.arange(n) % 32 == (9 if n > 32 else 1) if kind == "outlier" else np.arange(n) != 0
        if kind in ("outlier", "sink"):
            first = np.where(apart, -100, 100) if kind == "outlier" or c is pre else np.full(n, -100)
            if bits == 8:
                c[0][..., 0] = first
                c[1][:] = 0.02
            else:
                c[0][..., 0] = (c[0][..., 0] & 0xF0) | np.where(first > 0, 14, 1)  # (codes 96, -96)
                c[1][:] = np.float32(0.02).view(np.uint32) >> 16
        shape = c[3].shape
        size = np.ones(shape, np.float32)
        up = (slice(None), slice(None))
        if kind == "outlier":
            size[up + (apart,)] = 2.0 ** 30
        elif kind == "spread":
            size = (2.0 ** rng.uniform(-30, 30, shape)).astype(np.float32)
        elif kind == "sink":
            size[up + (slice(3, None, 7),)] = 0
            if c is pre:
                size[up + (0,)] = 2.0 ** -40
        elif kind == "blocks":
            size[..., -1] = 2.0 ** -44 if c is pre else 2.0 ** 44  # (int8: the last position's)
        else:
            size[up + (slice(0, 300 if n > 300 else 32),)] = 0
        v = (c[3] if bits == 8 else R.bf16(c[3])) * size
        c[3][:] = v if bits == 8 else (v.view(np.uint32) >> 16).astype(np.uint16)
    q = rng.standard_normal((beams, nq, hd))
    if kind in ("outlier", "sink"):  # some 30 between the scores of the two kinds of positions
        q[..., 0] = 60 * (hd / 64) ** 0.5
        q = R.unrotate(q)
    q = q.astype(np.float32)
    out = torch.full((beams, nq, hd), float("nan"), device="cuda")
    _, p = rows_of(pre, prefix)
    _, t = rows_of(tl, tail)
    ws = workspace(gpu_ctx.attn_shared_workspace(1, beams, nq, nkv, hd, prefix, tail))
    gpu_ctx.attn_shared(bits, dev(q.reshape(beams, -1)), nq * hd, 1, beams, nq, nkv, hd, p, t, hd ** -0.5, out, ws)
    gpu_ctx.sync()
    rows = list(range(beams)) if beams < 4 else [0, 31, 60]  # (the reference of a few rows)
    want, bound = R.attention(bits, q[rows], pre, [a[rows] for a in tl], [prefix], [tail] * len(rows), len(rows), nq, nkv, hd,
                              hd ** -0.5)
    err = np.abs(out.cpu().numpy()[rows] - want)
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("bits,hd", [(8, 64), (8, 128), (4, 64), (4, 128)])
@pytest.mark.parametrize("beams,nq,nkv,prefix,tail", [(3, 4, 2, 50, 20), (3, 4, 2, 1500, 200)])
@pytest.mark.parametrize("size", [1e3, 1e5, 1e7, 1e9, 1e13, 1e20])
def test_attention_of_scores_of_any_size(gpu_ctx, bits, hd, beams, nq, nkv, prefix, tail, size):
    """Scores from thousands to 1e20, where fp32 does not tell whole numbers apart: the best position of a head
    takes all the weight, and the output is its V."""
    rng = np.random.default_rng(hd + bits + prefix)
    pre, tl = R.new_cache(bits, 1, nkv, prefix, hd, rng), R.new_cache(bits, beams, nkv, tail, hd, rng)
    q = rng.standard_normal((beams, nq, hd)).astype(np.float32)
    scale = np.float32(size)
    out = torch.full((beams, nq, hd), float("nan"), device="cuda")
    _, p = rows_of(pre, prefix)
    _, t = rows_of(tl, tail)
    ws = workspace(gpu_ctx.attn_shared_workspace(1, beams, nq, nkv, hd, prefix, tail))
    gpu_ctx.attn_shared(bits, dev(q.reshape(beams, -1)), nq * hd, 1, beams, nq, nkv, hd, p, t, float(scale), out, ws)
    gpu_ctx.sync()
    got = out.cpu().numpy()
    import oracle as O
    pk, pv, tk, tv = (R.values(bits, *c) for c in (pre[:2], pre[2:], tl[:2], tl[2:]))
    told = 0
    for r in range(beams):
        for h in range(nq):
            g = h // (nq // nkv)
            code, qs = O.kv_quant_head(q[r, h])
            z = np.concatenate((pk[0, g], tk[r, g])) @ (code.astype(np.float64) * np.float64(qs)) * float(scale)
            first, second = np.sort(z)[[-1, -2]]
            # a score is off by 5 roundings: told apart beyond that, and by enough for the second to weigh nothing
            if first - second < 24 + 10 * R.U * max(first, -z.min()):
                continue
            told += 1
            v = np.concatenate((pv[0, g], tv[r, g]))[z.argmax()]
            # pieces of 2^-21, sums of one term, the rotation's 8 roundings
            bound = (2.0 ** -21 + 8 * R.U) * R.block_sums(np.abs(v)) / 8 + 2.0 ** -30
            assert (np.abs(got[r, h] - R.unrotate(v)) <= bound).all(), (r, h)
    assert told >= beams * nq // 2 and np.isfinite(got).all()


@pytest.mark.parametrize("bits,hd", [(8, 64), (8, 128), (4, 64), (4, 128)])
@pytest.mark.parametrize("prefix", [50, 1500])
@pytest.mark.parametrize("size", [3e8, 1e10, 1e14])
def test_attention_of_many_heads_with_scores_past_whole_numbers(gpu_ctx, bits, hd, prefix, size):
    """2048 heads whose scores' steps are 32 and more: whatever a step does to the largest score and to what it is
    referred to, its weight is not lost, and the head's output is its V."""
    beams, nq, nkv = 64, 32, 4
    rng = np.random.default_rng(hd + bits)
    pre = R.new_cache(bits, 1, nkv, prefix, hd, rng)
    q = rng.standard_normal((beams, nq, hd)).astype(np.float32)
    out = torch.full((beams, nq, hd), float("nan"), device="cuda")
    _, p = rows_of(pre, prefix)
    ws = workspace(gpu_ctx.attn_shared_workspace(1, beams, nq, nkv, hd, prefix, 0))
    gpu_ctx.attn_shared(bits, dev(q.reshape(beams, -1)), nq * hd, 1, beams, nq, nkv, hd, p, None, size, out, ws)
    gpu_ctx.sync()
    got = out.cpu().numpy()
    assert np.isfinite(got).all()
    import oracle as O
    code = np.stack([[c.astype(np.float64) * np.float64(s) for c, s in (O.kv_quant_head(h) for h in row)] for row in q])
    told = 0
    for g in range(nkv):
        k, v = (R.values(bits, pre[i][0, g], pre[i + 1][0, g]) for i in (0, 2))
        heads = slice(g * nq // nkv, (g + 1) * nq // nkv)
        z = (code[:, heads] @ k.T) * float(np.float32(size))
        first, second = np.moveaxis(np.sort(z, -1)[..., [-1, -2]], -1, 0)
        apart = first - second >= 24 + 10 * R.U * np.maximum(first, -z.min(-1))  # (as above)
        best = v[z.argmax(-1)]
        bound = (2.0 ** -21 + 8 * R.U) * R.block_sums(np.abs(best)) / 8 + 2.0 ** -30
        off = np.abs(got[:, heads] - R.unrotate(best))
        assert (off <= bound)[apart].all()
        told += int(apart.sum())
    assert told >= beams * nq * 3 // 4


@pytest.mark.parametrize("bits,hd", [(8, 128), (4, 64), (4, 128)])
@pytest.mark.parametrize("prefix", [50, 1500])
def test_attention_of_far_scores_stays_in_its_rows(gpu_ctx, bits, hd, prefix):
    """Infinite and enormous scores, and V scales far above or below, of one row's query or tail: the other
    rows' bits do not change."""
    rng = np.random.default_rng(prefix + 1)
    beams, nq, nkv, tail = 6, 8, 2, 20
    pre, tl = R.new_cache(bits, 1, nkv, prefix, hd, rng), R.new_cache(bits, beams, nkv, tail, hd, rng)
    q = rng.standard_normal((beams, nq * hd)).astype(np.float32)
    ws = workspace(gpu_ctx.attn_shared_workspace(1, beams, nq, nkv, hd, prefix, tail))

    def run():
        _, p = rows_of(pre, prefix)
        _, t = rows_of(tl, tail)
        out = torch.zeros((beams, nq, hd), device="cuda")
        gpu_ctx.attn_shared(bits, dev(q), nq * hd, 1, beams, nq, nkv, hd, p, t, hd ** -0.5, out, ws)
        gpu_ctx.sync()
        return out.cpu().numpy()

    def bf(v):
        return v if bits == 8 else np.float32(v).view(np.uint32) >> 16

    good = run()
    assert np.isfinite(good).all()
    q[1] *= 1e12
    q[2, 3 * hd:4 * hd] *= 1e30
    tl[1][3, 0, 7] = bf(np.inf)
    tl[3][4, 1, 2], tl[3][4, 0, 5] = bf(1e30), bf(1e-30)
    bad = run()
    assert np.array_equal(bad[[0, 5]], good[[0, 5]])
    assert np.array_equal(np.delete(bad[2], 3, 0), np.delete(good[2], 3, 0)) and np.isfinite(bad[1]).all()
    assert np.array_equal(bad[3, 4:], good[3, 4:])


def test_attention_agrees_with_attn_decode(gpu_ctx):
    """A row's output is the one-sequence operator's over its prefix and tail laid end to end."""
    rng = np.random.default_rng(11)
    beams, nq, nkv, hd, prefix, tail = 4, 8, 2, 128, 900, 61
    pre, tl = R.new_cache(8, 1, nkv, prefix, hd, rng), R.new_cache(8, beams, nkv, tail, hd, rng)
    q = (2 * rng.standard_normal((beams, nq, hd))).astype(np.float32)
    out = torch.empty((beams, nq, hd), device="cuda")
    _, p = rows_of(pre, prefix)
    _, t = rows_of(tl, tail)
    ws = workspace(gpu_ctx.attn_shared_workspace(1, beams, nq, nkv, hd, prefix, tail))
    gpu_ctx.attn_shared(8, dev(q.reshape(beams, -1)), nq * hd, 1, beams, nq, nkv, hd, p, t, hd ** -0.5, out, ws)
    _, bound = R.attention(8, q, pre, tl, [prefix], [tail] * beams, beams, nq, nkv, hd, hd ** -0.5)
    for r in range(beams):
        c = [dev(np.concatenate((a[0], b[r]), 1)) for a, b in zip(pre, tl)]
        one = torch.empty((nq, hd), device="cuda")
        gpu_ctx.attn_decode(8, dev(q[r]), nq, nkv, hd, *c, prefix + tail, prefix + tail, hd ** -0.5, one)
        # both are within the bound of the exact value
        assert (np.abs(out[r].cpu().numpy() - one.cpu().numpy()) <= 2 * bound[r]).all()


def test_attention_past_32_bit_offsets(gpu_ctx):
    """A prefix of 2^21 positions in a cache of 20 heads of 128 bytes (5 GiB), of which only the last
    100 positions matter: their scores are far above the others'."""
    hd, nkv, cap, beams = 128, 20, 1 << 21, 2
    kq = torch.zeros(nkv * cap, hd, dtype=torch.int8, device="cuda")
    ks = torch.full((nkv * cap,), 0.05, device="cuda")
    rng = np.random.default_rng(3)
    tail = R.new_cache(8, 1, nkv, 100, hd, rng)
    q = (4 * rng.standard_normal((beams, nkv, hd))).astype(np.float32)
    import oracle as O
    for h in range(nkv):
        code = O.kv_quant_head(q[0, h])[0].astype(np.int64)
        tail[0][0, h] = np.clip(code + rng.integers(-20, 21, (100, hd)), -127, 127)
        tail[1][0, h] = 0.05
        at = slice((h + 1) * cap - 100, (h + 1) * cap)
        kq[at], ks[at] = dev(tail[0][0, h]), dev(tail[1][0, h])
    q[1] = q[0]
    p = k2t.KVRows(kq, ks, kq, ks, cap=cap)  # (V is K)
    out = torch.empty((beams, nkv, hd), device="cuda")
    ws = workspace(gpu_ctx.attn_shared_workspace(1, beams, nkv, nkv, hd, cap, 0))
    gpu_ctx.attn_shared(8, dev(q.reshape(beams, -1)), nkv * hd, 1, beams, nkv, nkv, hd, p, None, 1.0, out, ws)
    gpu_ctx.sync()
    tail[2], tail[3] = tail[0], tail[1]
    none = R.new_cache(8, 1, nkv, 1, hd, rng)
    both = [np.repeat(a, beams, 0) for a in tail]
    want, bound = R.attention(8, q, none, both, [0], [100] * beams, beams, nkv, nkv, hd, 1.0)
    err = np.abs(out.cpu().numpy() - want)
    assert (err <= 2 * bound).all(), float((err / bound).max())


# ---------------------------------------------------------------- select
def run_select(ctx, logits, scores, done, n_seq, beams, k, eos, stride=None):
    v = logits.shape[1]
    wide = np.full((logits.shape[0], stride or v), 1e30, np.float32)
    wide[:, :v] = logits
    n = (n_seq, k)
    o = [torch.full(n, -7, dtype=d, device="cuda") for d in (torch.float32, torch.int32, torch.int32, torch.int32)]
    ws = workspace(ctx.beam_select_workspace(n_seq, beams, v, k))
    ctx.beam_select(dev(wide), v, wide.shape[1], dev(scores), None if done is None else dev(done), n_seq, beams, k, eos,
                    *o, ws)
    ctx.sync()
    return [t.cpu().numpy() for t in o]


# exp is off by 4 units and by a rounding of its exponent, of which 18 bits count in a sum of up to 2^18
# terms (18 ln 2 2^-24 < 2^-20); a sum of 4096 in lanes, waves and slices by 40 roundings: the logarithm
# by less than 2^-18; the score is then rounded once
def score_tol(s):
    return np.where(np.isfinite(s), np.abs(s) * R.U, 0) + 2.0 ** -18


@pytest.mark.parametrize("n_seq,beams,vocab,k", [(1, 1, 1, 1), (1, 1, 7, 9), (1, 4, 8192, 4), (3, 2, 1001, 128), (2, 8, 4097, 16),
                                                 (1, 64, 515, 128), (1, 5, 49152, 10), (2, 3, 20000, 1)])
@pytest.mark.parametrize("with_done", [False, True])
def test_select_matches_the_reference(gpu_ctx, n_seq, beams, vocab, k, with_done):
    print(f"beam_select {n_seq} {beams} {vocab} {k} done={with_done}", flush=True)
    rng = np.random.default_rng(vocab + k)
    rows = n_seq * beams
    logits = (3 * rng.standard_normal((rows, vocab))).astype(np.float32)
    scores = rng.uniform(-9, -1, rows).astype(np.float32)
    eos = min(3, vocab - 1)
    done = (rng.random(rows) < 0.4).astype(np.int32) if with_done else None
    if beams > 2:
        scores[1] = -np.inf  # a row not in use, whose logits mean nothing
        logits[1] = np.nan
    ws, wt, wp, wd, gap = R.select(logits, scores, done, n_seq, beams, k, eos)
    assert gap > 2.0 ** -15, "inputs too near a tie to be told apart"
    s, t, p, d = run_select(gpu_ctx, logits, scores, done, n_seq, beams, k, eos, stride=vocab + 5)
    assert np.array_equal(t, wt) and np.array_equal(p, wp) and np.array_equal(d, wd)
    assert np.array_equal(np.isinf(s), np.isinf(ws)) and (np.abs(s - ws)[np.isfinite(ws)] <= score_tol(ws)[np.isfinite(ws)]).all()


def test_select_ties_masks_and_odd_values(gpu_ctx):
    """Equal logits and equal rows (the lower token, the lower row first), -inf and NaN logits, rows
    of the lowest value, +inf, a row with nothing, few candidates."""
    v, k = 5000, 12
    base = np.zeros((6, v), np.float32)
    base[1] = base[0]  # two equal rows of equal logits
    base[2] = np.finfo(np.float32).min  # a mask of the lowest value everywhere
    base[3] = -np.inf
    base[3, [4999, 17, 4096]] = [1.0, 1.0, np.nan]
    base[4] = -np.inf
    base[5, 4321] = np.inf
    base[5, 7] = -0.0
    cases = [([-1, -1, -20, -20, -20, -20], 6), ([-9, -9, -1, -9, -9, -9], 6), ([-np.inf] * 3 + [-2, -1, -np.inf], 6),
             ([-50, -50, -50, -50, -50, 0], 6), ([np.nan, -np.inf, -np.inf, 0, 0, -np.inf], 6)]
    for scores, beams in cases:
        sc = np.array(scores, np.float32)
        ws, wt, wp, wd, _ = R.select(base, sc, None, 1, beams, k, 17)
        s, t, p, d = run_select(gpu_ctx, base, sc, None, 1, beams, k, 17)
        assert np.array_equal(t, wt) and np.array_equal(p, wp) and np.array_equal(d, wd), scores
        w32 = ws.astype(np.float32)
        fin = np.isfinite(w32)
        assert np.array_equal(s[~fin], w32[~fin]) and (np.abs(s - ws)[fin] <= score_tol(ws)[fin]).all(), scores


def test_select_joins_slices_in_64_bits(gpu_ctx):
    """One logit in every 4096, so that no fp32 sum has two terms: rows whose scores are 2^-45 apart come in
    order. (A row's score so far is the fp32 next to its log-sum, so that all the best ones are next to zero.)"""
    rng = np.random.default_rng(12)
    beams, slices = 48, 9
    logits = np.full((beams, 4096 * slices), -np.inf, np.float32)
    lse = np.empty(beams)
    for r in range(beams):
        x = rng.uniform(-3, 0, slices).astype(np.float32)
        x[rng.integers(slices)] = 0
        logits[r, np.arange(slices) * 4096 + rng.integers(0, 4096, slices)] = x
        lse[r] = np.log(np.exp(x.astype(np.float64)).sum())
    scores = lse.astype(np.float32)
    ws, wt, wp, wd, gap = R.select(logits, scores, None, 1, beams, beams, -1)
    assert gap > 2.0 ** -45 and len(set(wp[0])) == beams  # (one candidate of every row; 64 bits' own roundings: 2^-50)
    s, t, p, d = run_select(gpu_ctx, logits, scores, None, 1, beams, beams, -1)
    assert np.array_equal(t, wt) and np.array_equal(p, wp) and np.array_equal(d, wd)
    assert (np.abs(s - ws) <= np.abs(ws) * R.U + 2.0 ** -50).all()


@pytest.mark.parametrize("order", ["rising", "falling", "blocks", "equal"])
def test_select_of_ordered_logits(gpu_ctx, order):
    """The k best all in one place, or all equal: the same choice however the slices are cut."""
    v, k = 9000, 100
    x = np.arange(v, dtype=np.float32) / 64
    if order == "falling":
        x = x[::-1].copy()
    elif order == "blocks":
        x = (np.arange(v) % 64 // 4).astype(np.float32)
    elif order == "equal":
        x[:] = 2.5
    logits, scores = np.stack((x, x, x)), np.array([-3, -2, -2], np.float32)
    ws, wt, wp, wd, _ = R.select(logits, scores, None, 1, 3, k, -1)
    s, t, p, d = run_select(gpu_ctx, logits, scores, None, 1, 3, k, -1)
    assert np.array_equal(t, wt) and np.array_equal(p, wp) and np.array_equal(d, wd)
    assert (np.abs(s - ws) <= score_tol(ws)).all()


def test_select_in_place_and_without_flags(gpu_ctx):
    """k == beams: the scores and done flags are replaced in place; done flags may be left out."""
    rng = np.random.default_rng(9)
    n, beams, v = 3, 4, 700
    logits = rng.standard_normal((n * beams, v)).astype(np.float32)
    scores, done = rng.uniform(-5, 0, n * beams).astype(np.float32), (rng.random(n * beams) < 0.3).astype(np.int32)
    ws, wt, wp, wd, gap = R.select(logits, scores, done, n, beams, beams, 1)
    assert gap > 2.0 ** -15
    ds, dd = dev(scores), dev(done)
    tok, par = ints([0] * n * beams), ints([0] * n * beams)
    w = workspace(gpu_ctx.beam_select_workspace(n, beams, v, beams))
    gpu_ctx.beam_select(dev(logits), v, v, ds, dd, n, beams, beams, 1, ds, tok, par, dd, w)
    gpu_ctx.sync()
    assert np.array_equal(tok.cpu().numpy(), wt.reshape(-1)) and np.array_equal(par.cpu().numpy(), wp.reshape(-1))
    assert np.array_equal(dd.cpu().numpy(), wd.reshape(-1))
    assert (np.abs(ds.cpu().numpy() - ws.reshape(-1)) <= score_tol(ws.reshape(-1))).all()
    gpu_ctx.beam_select(dev(logits), v, v, dev(scores), None, n, beams, beams, -1, ds, tok, par, None, w)
    gpu_ctx.sync()
    _, wt, wp, _, _ = R.select(logits, scores, None, n, beams, beams, -1)
    assert np.array_equal(tok.cpu().numpy(), wt.reshape(-1)) and np.array_equal(par.cpu().numpy(), wp.reshape(-1))


@pytest.mark.parametrize("vocab,k,spread", [(100000, 128, True), (5000, 64, False)])
def test_select_of_64_rows(gpu_ctx, vocab, k, spread):
    """More candidates than the merge holds: every third slice far above the others, so that a row has
    hundreds beyond its bound; all logits and rows equal, so that every candidate reaches the last one."""
    rng = np.random.default_rng(vocab)
    logits, scores = np.full((64, vocab), 0.75, np.float32), np.full(64, -2.0, np.float32)
    if spread:
        high = np.arange(vocab) // 4096 % 3 == 1
        for r in range(64):  # (the same values in every row: scores 2^-13 apart tell the rows apart)
            logits[r, high] = 600 + rng.permutation(high.sum()) / 128
            logits[r, ~high] = rng.permutation((~high).sum()) / 256
        scores = (-3 - np.arange(64) / 2.0 ** 13).astype(np.float32)
    ws, wt, wp, wd, gap = R.select(logits, scores, None, 1, 64, k, 11)
    assert gap > 2.0 ** -15 or not spread
    s, t, p, d = run_select(gpu_ctx, logits, scores, None, 1, 64, k, 11)
    assert np.array_equal(t, wt) and np.array_equal(p, wp) and np.array_equal(d, wd)
    assert (np.abs(s - ws) <= score_tol(ws)).all()


def test_the_most_rows(gpu_ctx):
    """65535 rows in one call of each kind, of one position each: the attention is then the V head read
    back, a rearrangement permutes what is read back, a choice is the sorted sums."""
    beams, n_seq, nkv, hd = 15, 4369, 2, 64
    rows = n_seq * beams
    assert rows == 65535
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(rows, 6 * hd, generator=g, device="cuda")  # 2 query, 2 K, 2 V heads
    codes = [torch.zeros(rows, nkv, 1, hd, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.zeros(rows, nkv, 1, device="cuda") for _ in range(2)]
    kv = k2t.KVRows(codes[0], scales[0], codes[1], scales[1], cap=1)
    zero = torch.zeros(rows, dtype=torch.int32, device="cuda")

    def load():
        k, v = torch.zeros(rows, nkv, hd, device="cuda"), torch.zeros(rows, nkv, hd, device="cuda")
        gpu_ctx.kv_load(8, kv, rows, 1, nkv, hd, zero, k, v, nkv * hd)
        gpu_ctx.sync()
        return k, v

    at = x.data_ptr()
    gpu_ctx.kv_append(8, at + 8 * hd, at + 16 * hd, 6 * hd, rows, 1, nkv, hd, zero, kv)
    k, v = load()
    # a code is off by half a step of max |r| / 127, and max |r| <= sqrt(64) max |x|; the rotation sums 64
    assert (v - x[:, 4 * hd:].view(rows, nkv, hd)).abs().max() <= 8 * 8 * x.abs().max() / 254
    out = torch.full((rows, nkv, hd), float("nan"), device="cuda")
    ws = workspace(gpu_ctx.attn_shared_workspace(n_seq, beams, nkv, nkv, hd, 0, 1))
    gpu_ctx.attn_shared(8, x, 6 * hd, n_seq, beams, nkv, nkv, hd, None, kv, 0.125, out, ws)
    gpu_ctx.sync()
    assert (out - v).abs().max() <= 2.0 ** -18 * v.abs().max()
    parents = torch.arange(rows, dtype=torch.int32, device="cuda").view(n_seq, beams).flip(1).contiguous()
    gpu_ctx.kv_reorder(8, kv, parents, 1, n_seq, beams, nkv, hd)
    k2, v2 = load()
    assert torch.equal(k2, k[parents.view(-1).long()]) and torch.equal(v2, v[parents.view(-1).long()])
    logits, scores = torch.randn(rows, 3, generator=g, device="cuda"), torch.randn(rows, generator=g, device="cuda")
    o = [torch.zeros(n_seq, 7, dtype=d, device="cuda") for d in (torch.float32, torch.int32, torch.int32)]
    ws = workspace(gpu_ctx.beam_select_workspace(n_seq, beams, 3, 7))
    gpu_ctx.beam_select(logits, 3, 3, scores, None, n_seq, beams, 7, -1, *o, None, ws)
    gpu_ctx.sync()
    cand = scores.double()[:, None] + torch.log_softmax(logits.double(), 1)
    want = cand.view(n_seq, -1).sort(1, descending=True).values[:, :7]
    assert (o[0] - want).abs().max() <= 2.0 ** -18 + 2.0 ** -24 * want.abs().max()
    chosen = cand[o[2].long(), o[1].long()]  # and the token and row named have that score
    assert (chosen - want).abs().max() <= 2.0 ** -18
    assert (o[2] // beams == torch.arange(n_seq, device="cuda")[:, None]).all()


@pytest.mark.parametrize("bits,hd", [(8, 64), (8, 128), (4, 64), (4, 128)])
@pytest.mark.parametrize("beams,prefix,tail", [(3, 60, 9), (8, 1500, 40), (64, 900, 300)])
@pytest.mark.parametrize("size", [2.9e6, 1.1e7, 3e7, 1e9, 1e13])
def test_attention_of_far_scores_with_v_scales_far_apart(gpu_ctx, bits, hd, beams, prefix, tail, size):
    """Scores of 2.9e6 (2^22 powers of two) to 1e13 and V scales 2^-30 .. 2^30: a large scale of small weight takes
    nothing from the best position's V."""
    nq, nkv = 8, 2
    g = nq // nkv
    rng = np.random.default_rng(hd + bits + prefix)
    pre, tl = R.new_cache(bits, 1, nkv, prefix, hd, rng), R.new_cache(bits, beams, nkv, tail, hd, rng)
    for c in (pre, tl):
        f = np.exp2(rng.uniform(-30, 30, c[3].shape)).astype(np.float32)
        c[3][:] = f if bits == 8 else (f.view(np.uint32) >> 16).astype(np.uint16)
    q = rng.standard_normal((beams, nq, hd)).astype(np.float32)
    scale = np.float32(size / (4 * 2 * hd ** 0.5))  # (|q . k| is about 2 sqrt(hd) at one standard deviation)
    out = torch.full((beams, nq, hd), float("nan"), device="cuda")
    _, p = rows_of(pre, prefix)
    _, t = rows_of(tl, tail)
    ws = workspace(gpu_ctx.attn_shared_workspace(1, beams, nq, nkv, hd, prefix, tail))
    gpu_ctx.attn_shared(bits, dev(q.reshape(beams, -1)), nq * hd, 1, beams, nq, nkv, hd, p, t, float(scale), out, ws)
    gpu_ctx.sync()
    got = out.cpu().numpy()
    assert np.isfinite(got).all()
    import oracle as O
    told = 0
    for r in range(beams):
        for h in range(nkv):
            k, v, s = (np.concatenate((f(pre)[0, h], f(tl)[r, h])) for f in (
                lambda c: R.values(bits, c[0], c[1]), lambda c: R.values(bits, c[2], c[3]),
                lambda c: np.log2((c[3] if bits == 8 else R.bf16(c[3])).astype(np.float64)).reshape(c[3].shape[:3] + (-1,))))
            x = np.stack([c.astype(np.float64) * np.float64(e) for c, e in (O.kv_quant_head(a) for a in q[r, h * g:(h + 1) * g])])
            z = (x @ k.T) * float(scale)
            best = z.argmax(1)
            # a score is off by 5 roundings of the largest; the others weigh 2^-45 at most, next to their V scales
            gap = z.max(1, keepdims=True) - z - 10 * R.U * np.abs(z).max(1, keepdims=True)
            gap -= np.log(2) * (45 + np.maximum((s[None] - s[best][:, None]).max(-1), 0))
            gap[np.arange(g), best] = np.inf
            ok = gap.min(1) >= 0
            bound = (2.0 ** -21 + 8 * R.U + 2.0 ** -30) * R.block_sums(np.abs(v[best])) / 8
            assert (np.abs(got[r, h * g:(h + 1) * g] - R.unrotate(v[best])) <= bound)[ok].all(), (r, h)
            told += int(ok.sum())
    assert told >= 0.6 * beams * nq


@pytest.mark.parametrize("beams,prefix,tail", [(3, 60, 9), (8, 1500, 40)])
@pytest.mark.parametrize("first,second", [(2.0 ** 20, 0.0), (2.0 ** 60, 0.0), (0.0, 2.0 ** 60), (2.0 ** 25, 2.0 ** -80), (0.0, 0.0)])
def test_attention_of_nf4_blocks_of_scales_far_apart(gpu_ctx, beams, prefix, tail, first, second):
    """The two V blocks of a head of 128: one of zeros, or one 2^105 times the other."""
    nq, nkv, hd = 8, 2, 128
    rng = np.random.default_rng(prefix)
    pre, tl = R.new_cache(4, 1, nkv, prefix, hd, rng), R.new_cache(4, beams, nkv, tail, hd, rng)
    for c in (pre, tl):
        for b, size in ((0, first), (1, second)):
            f = (rng.uniform(1, 2, c[3].shape[:3]) * size).astype(np.float32)
            c[3][..., b] = (f.view(np.uint32) >> 16).astype(np.uint16)
    q = rng.standard_normal((beams, nq, hd)).astype(np.float32)
    out = torch.full((beams, nq, hd), float("nan"), device="cuda")
    _, p = rows_of(pre, prefix)
    _, t = rows_of(tl, tail)
    ws = workspace(gpu_ctx.attn_shared_workspace(1, beams, nq, nkv, hd, prefix, tail))
    gpu_ctx.attn_shared(4, dev(q.reshape(beams, -1)), nq * hd, 1, beams, nq, nkv, hd, p, t, 0.17, out, ws)
    gpu_ctx.sync()
    want, bound = R.attention(4, q, pre, tl, [prefix], [tail] * beams, beams, nq, nkv, hd, 0.17)
    assert (np.abs(out.cpu().numpy() - want) <= bound).all()


@pytest.mark.parametrize("hd,nq,nkv,tail", [(64, 2, 2, 1), (128, 8, 2, 1), (64, 32, 8, 900)])
def test_attention_of_one_position_rounds_its_v_to_nearest(gpu_ctx, hd, nq, nkv, tail):
    """Zero queries, one position, and a V head of a single code 1: what comes out is the V scale over 8, every step exact
    but for the scale's two pieces, 2^-23 of it, and their sum, a step at most."""
    beams = 60
    rng = np.random.default_rng(hd + nq)
    tl = R.new_cache(8, beams, nkv, tail, hd, rng)
    tl[2][:] = 0
    at = rng.integers(0, hd, (beams, nkv, 1))
    np.put_along_axis(tl[2], np.broadcast_to(at, tl[3].shape)[..., None], 1, -1)
    tl[3][:] = rng.uniform(2.0 ** -6, 2.0 ** -3, (beams, nkv, 1))
    out = torch.full((beams, nq, hd), float("nan"), device="cuda")
    _, t = rows_of(tl, tail, d_len=ints([1] * beams))
    ws = workspace(gpu_ctx.attn_shared_workspace(1, beams, nq, nkv, hd, 0, tail))
    gpu_ctx.attn_shared(8, torch.zeros(beams, nq * hd, device="cuda"), nq * hd, 1, beams, nq, nkv, hd, None, t, 0.17, out, ws)
    gpu_ctx.sync()
    got = out.cpu().numpy()
    vs = np.repeat(tl[3][:, :, 0].astype(np.float64), nq // nkv, 1)[..., None]
    where = np.repeat(at[..., 0], nq // nkv, 1)[..., None] // 64 == np.arange(hd) // 64
    assert (got[~where] == 0).all()
    off = (np.abs(np.abs(got) * 8 - vs) / vs)[where]
    assert off.max() <= 2.0 ** -23 + 2.0 ** -23, off.max()
