"""Blocks of tokens: rotary positions (k2t_rope), attention over the rows' caches (k2t_attn_tokens), adjustments of
logits (k2t_logits_adjust) and the positions that a cache keeps (k2t_kv_keep), against 64-bit references (block_ref) and the
one-token operators."""

import numpy as np
import pytest
import torch

import block_ref as R
import branch_ref as B
import k2t
from test_block_args import KINDS
from test_gpu_branch import dev, host, ints, rows_of, workspace

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- rope
@pytest.mark.parametrize("hd,rot,interleaved,kind", [
    (64, 64, False, "plain"), (64, 64, True, "plain"), (128, 128, False, "ramp"), (128, 128, True, "wave"), (128, 64, False, "linear"),
    (128, 40, True, "base"), (64, 32, False, "plain"), (64, 8, True, "plain"), (128, 90, False, "plain"), (128, 66, True, "ramp"),
    (64, 2, False, "plain"), (64, 2, True, "plain"), (64, 12, False, "wave"), (64, 62, True, "linear")])
@pytest.mark.parametrize("batch,ntok,heads,in_place", [(1, 1, 1, False), (3, 7, 5, True), (4, 1, 12, False), (2, 130, 3, True), (37, 60, 2, False)])
def test_rope(gpu_ctx, hd, rot, interleaved, kind, batch, ntok, heads, in_place):
    print(f"rope hd={hd} rot={rot} interleaved={interleaved} {kind} batch={batch} ntok={ntok} heads={heads}", flush=True)
    rng = np.random.default_rng(hd * rot + batch * ntok)
    theta = 100000.0
    plan = k2t.RopePlan(int(interleaved), rot, theta, KINDS[kind], 16.0, 8192)
    turn, scale = R.turns(rot, theta, kind, 16.0, 8192)
    xs, os_ = heads * hd + 8, heads * hd + (8 if in_place else 4)
    x = (rng.standard_normal((batch * ntok, xs)) * rng.uniform(0.01, 9, (batch * ntok, 1))).astype(np.float32)
    pos = rng.integers(-5, 200000, batch).astype(np.int32)
    pos[0] = 0
    if batch > 1:
        pos[1] = 2 ** 31 - 1
    counts = rng.integers(0, ntok + 3, batch).astype(np.int32)
    counts[0] = ntok
    depth = rng.integers(0, ntok, (batch, ntok)).astype(np.int32) if ntok > 1 and batch % 2 else None
    at = pos.astype(np.int64)[:, None] + (np.arange(ntok) if depth is None else depth)
    dx = dev(x)
    out = dx if in_place else torch.full((batch * ntok, os_), 3.25, device="cuda")
    gpu_ctx.rope(dx, xs, batch, ntok, heads, hd, dev(pos), plan, out, os_, depth=None if depth is None else dev(depth), counts=dev(counts))
    gpu_ctx.sync()
    got = out.cpu().numpy()
    want, bound = R.rope(x[:, :heads * hd].reshape(-1, heads, hd), at.reshape(-1), turn, scale, interleaved)
    if not in_place:
        assert np.array_equal(dx.cpu().numpy(), x)
    live = (np.arange(ntok) < counts[:, None]).reshape(-1)
    rest = x if in_place else np.full((batch * ntok, os_), 3.25, np.float32)
    assert np.array_equal(got[~live], rest[~live]) and np.array_equal(got[:, heads * hd:], rest[:, heads * hd:])
    y = got[live][:, :heads * hd].reshape(-1, heads, hd)
    assert np.array_equal(y[..., rot:], x[live][:, :heads * hd].reshape(-1, heads, hd)[..., rot:])
    assert (np.abs(y - want[live]) <= bound[live]).all()


def test_rope_agrees_with_the_models_table(gpu_ctx):
    """The oracle's rotation (the reference's fp32 table): its angles are fp32 products, off by up to 2^-24 p."""
    import oracle as O
    rng = np.random.default_rng(3)
    hd, pos = 64, np.array([0, 1, 17, 400, 2047], np.int32)
    x = rng.standard_normal((5, hd)).astype(np.float32)
    want = np.stack([O.rope_apply(x[i], O.rope_row(hd, 100000.0, int(p))) for i, p in enumerate(pos)])
    out = torch.zeros(5, hd, device="cuda")
    gpu_ctx.rope(dev(x), hd, 5, 1, 1, hd, dev(pos), k2t.RopePlan(k2t.ROPE_HALF, hd, 100000.0), out, hd)
    gpu_ctx.sync()
    tol = (8 + 4 * pos[:, None]) * R.U * 2 * np.abs(x).max()
    assert (np.abs(out.cpu().numpy() - want) <= tol).all()


def test_rope_keeps_odd_values_in_their_pairs(gpu_ctx):
    x = np.ones((3, 128), np.float32)
    x[1, 5], x[1, 64 + 9], x[2, 70] = np.nan, np.inf, np.nan
    out = torch.zeros(3, 128, device="cuda")
    gpu_ctx.rope(dev(x), 128, 1, 3, 2, 64, ints([7]), k2t.RopePlan(k2t.ROPE_HALF, 32, 1e4), out, 128)
    gpu_ctx.sync()
    bad = ~np.isfinite(out.cpu().numpy())
    want = np.zeros((3, 128), bool)
    want[1, [5, 21, 64 + 9, 64 + 25]] = True
    want[2, [70, 86]] = True
    assert np.array_equal(bad, want)


# ---------------------------------------------------------------- attention
def tree(rng, ntok):
    sees = np.zeros(ntok, np.uint64)
    for t in range(ntok):
        sees[t] = np.uint64(1 << t) | (sees[rng.integers(max(0, t - 4), t)] if t else np.uint64(0))
    return sees


def attend(ctx, bits, q, cache, pos, counts, sees, nq, nkv, hd, scale, length, extra=0):
    """k2t_attn_tokens with q rows 8 floats apart, guarded output and workspace, and the workspace's own size."""
    batch, ntok = q.shape[:2]
    wide = np.full((batch * ntok, nq * hd + 8), np.nan, np.float32)
    wide[:, :nq * hd] = q.reshape(batch * ntok, -1)
    t, kv = rows_of(cache, cache[0].shape[2], length=length)
    n = ctx.attn_tokens_workspace(batch, ntok, nq, nkv, hd, length + extra)
    ws = torch.full((n + 64,), 0x7F, dtype=torch.uint8, device="cuda")
    out = torch.full((batch * ntok + 1, nq * hd), 3.25, device="cuda")
    ctx.attn_tokens(bits, dev(wide), nq * hd + 8, batch, ntok, nq, nkv, hd, dev(pos), kv, scale, out, ws[:n],
                    counts=None if counts is None else dev(counts), sees=None if sees is None else dev(sees.view(np.int64)))
    ctx.sync()
    assert (ws[n:] == 0x7F).all() and (out[-1] == 3.25).all()
    for g, w in zip(t, cache):
        assert host(g, w).tobytes() == w.tobytes()
    return out[:-1].cpu().numpy().reshape(batch, ntok, nq, hd)


def check(got, want, bound):
    gone = np.isnan(bound)
    assert (got[gone] == 3.25).all()
    off = np.abs(got - want)
    ok = (off <= bound) | gone
    assert ok.all(), (np.argwhere(~ok)[:4], got[~ok][:4], want[~ok][:4], bound[~ok][:4], (off / bound)[~gone].max())


def case(rng, bits, batch, ntok, nq, nkv, hd, start, with_counts, with_tree, spare=3, first=None):
    cap = start + ntok + spare
    cache = B.new_cache(bits, batch, nkv, cap, hd, rng)
    q = rng.standard_normal((batch, ntok, nq, hd)).astype(np.float32)
    pos = rng.integers(max(0, start - 20), start + 1, batch).astype(np.int32)
    pos[0] = start
    counts = np.full(batch, ntok, np.int32)
    if with_counts:
        counts = rng.integers(0, ntok + 2, batch).astype(np.int32)
        counts[-1] = (ntok + 1) // 2
    if first is not None:  # row 0: all of its tokens, from this position on
        pos[0], counts[0] = first, ntok
    sees = np.stack([tree(rng, ntok) for _ in range(batch)]) if with_tree else None
    # what lies behind a row's block is never read: NaN scales
    for r in range(batch):
        end = pos[r] + max(0, min(counts[r], ntok))
        for a in (cache[1], cache[3]):
            a[r, :, end:] = np.nan if bits == 8 else 0x7FC0
    return q, cache, pos, counts if with_counts else None, sees, cap


HEADS = [(1, 1), (4, 2), (9, 3), (3, 3), (8, 1), (40, 2)]


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("i,batch,ntok,start,with_counts,with_tree", [
    (0, 1, 1, 0, False, False), (1, 2, 1, 33, False, False), (2, 1, 2, 0, False, False), (3, 3, 5, 31, True, True), (4, 2, 16, 64, True, False),
    (5, 1, 17, 5, False, True), (0, 4, 33, 0, True, False), (1, 1, 64, 130, False, True), (2, 2, 65, 3, True, False), (0, 1, 63, 1, False, True),
    (3, 1, 130, 64, False, False), (4, 1, 40, 300, False, True), (1, 1, 257, 0, False, False), (2, 1, 10, 700, False, True), (0, 2, 3, 1500, True, True),
    (5, 1, 2, 257, False, False), (4, 1, 150, 127, True, False), (2, 1, 1, 2500, False, False)])
def test_attention_of_blocks(gpu_ctx, bits, hd, i, batch, ntok, start, with_counts, with_tree):
    nq, nkv = HEADS[i]
    print(f"attn_tokens bits={bits} hd={hd} heads={nq}/{nkv} batch={batch} ntok={ntok} start={start} tree={with_tree}", flush=True)
    rng = np.random.default_rng(bits * hd + ntok * 7 + start)
    q, cache, pos, counts, sees, cap = case(rng, bits, batch, ntok, nq, nkv, hd, start, with_counts, with_tree)
    want, bound = R.attention(bits, q, cache, pos, np.full(batch, ntok) if counts is None else counts, sees, nq, nkv, hd, 0.17, cap)
    got = attend(gpu_ctx, bits, q, cache, pos, counts, sees, nq, nkv, hd, 0.17, cap, extra=ntok)
    check(got, want, bound)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd,nq,nkv,ntok,start", [(64, 2, 1, 9, 40), (128, 8, 2, 20, 300), (128, 2, 2, 64, 1300), (64, 16, 1, 64, 90)])
def test_attention_masks_that_leave_nothing(gpu_ctx, bits, hd, nq, nkv, ntok, start):
    """Rows whose tokens see nothing, bits of tokens that a row does not have, all bits, positions outside the cache, and a
    cache that ends inside the block."""
    rng = np.random.default_rng(ntok + start)
    batch = 6
    q, cache, pos, _, _, cap = case(rng, bits, batch, ntok, nq, nkv, hd, start, False, False)
    sees = np.zeros((batch, ntok), np.uint64)
    counts = np.full(batch, ntok, np.int32)
    full = np.uint64(0xFFFFFFFFFFFFFFFF)
    pos[:] = [0, start, 0, start, -2, start]
    sees[1] = full
    sees[2] = full  # of a row that has four of its tokens
    counts[2] = 4
    sees[3, ::3] = 1  # some tokens of a block see its first
    sees[4] = full
    sees[5] = np.uint64(2)
    for r in range(batch):
        for a in (cache[1], cache[3]):
            a[r] = rng.uniform(0.005, 0.05, a[r].shape).astype(np.float32) if bits == 8 else 0x3C23
    for length in (cap, start + 2, min(3, start)):
        want, bound = R.attention(bits, q, cache, pos, counts, sees, nq, nkv, hd, 0.2, length)
        check(attend(gpu_ctx, bits, q, cache, pos, counts, sees, nq, nkv, hd, 0.2, length), want, bound)
        want, bound = R.attention(bits, q, cache, pos, counts, None, nq, nkv, hd, 0.2, length)
        check(attend(gpu_ctx, bits, q, cache, pos, counts, None, nq, nkv, hd, 0.2, length), want, bound)
    empty = attend(gpu_ctx, bits, q, cache, pos, counts, None, nq, nkv, hd, 0.2, 0)
    assert (empty[counts == ntok] == 0).all()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd,nq,nkv,ntok,start", [(64, 2, 2, 12, 50), (128, 8, 1, 64, 200), (128, 4, 4, 150, 0), (64, 3, 1, 40, 1100)])
def test_attention_of_bad_positions_stays_where_they_are_seen(gpu_ctx, bits, hd, nq, nkv, ntok, start):
    """NaN and infinite scales of a token of the block reach the tokens that see it and no other; a NaN query its own heads."""
    rng = np.random.default_rng(ntok)
    q, cache, pos, counts, sees, cap = case(rng, bits, 2, ntok, nq, nkv, hd, start, False, ntok <= 64)
    clean, bound = R.attention(bits, q, cache, pos, np.full(2, ntok), sees, nq, nkv, hd, 0.2, cap)
    bad_t, bad_q = ntok // 2, ntok - 1
    see = [R.visible(ntok, int(pos[r]), ntok, cap, None if sees is None else [int(x) for x in sees[r]]) for r in range(2)]
    for which, value in ((1, "nan"), (3, "nan"), (3, "inf"), (1, "inf")):
        c = [a.copy() for a in cache]
        v = {8: {"nan": np.nan, "inf": np.inf}, 4: {"nan": 0x7FC0, "inf": 0x7F80}}[bits][value]
        c[which][0, :, pos[0] + bad_t] = v
        x = q.copy()
        x[1, bad_q, 0] = np.nan
        got = attend(gpu_ctx, bits, x, c, pos, None, sees, nq, nkv, hd, 0.2, cap)
        untouched = np.ones((2, ntok, nq), bool)
        untouched[0, see[0][:, pos[0] + bad_t]] = False
        untouched[1, bad_q, 0] = False
        assert np.isfinite(got[untouched]).all()
        assert (np.abs(got - clean)[untouched] <= bound[untouched]).all()
        if value == "nan":
            assert np.isnan(got[0][see[0][:, pos[0] + bad_t]]).any(-1).all()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd,nq,nkv,ntok,start", [(64, 2, 1, 3, 400), (128, 8, 2, 40, 100), (128, 2, 2, 150, 0)])
@pytest.mark.parametrize("kind", ["large", "peaked", "vscales", "small", "zero"])
def test_attention_of_values_of_any_size(gpu_ctx, bits, hd, nq, nkv, ntok, start, kind):
    """Scores of any size (K scales), V scales 2^80 apart, zero queries."""
    rng = np.random.default_rng(hd + ntok)
    q, cache, pos, counts, sees, cap = case(rng, bits, 1, ntok, nq, nkv, hd, start, False, False)
    end = start + ntok
    shape = cache[1][0, :, :end].shape

    def scales(lo, hi):
        f = np.exp2(rng.uniform(lo, hi, shape)).astype(np.float32)
        return f if bits == 8 else (f.view(np.uint32) >> 16).astype(np.uint16)
    if kind == "large":
        cache[1][0, :, :end] = scales(4, 6)
    elif kind == "peaked":
        cache[1][0, :, :end] = scales(-2, 1)
    elif kind == "vscales":
        cache[3][0, :, :end] = scales(-60, 20)
    elif kind == "small":
        cache[3][0, :, :end] = scales(-95, -90)
    else:
        q[0, ::2] = 0.0
    want, bound = R.attention(bits, q, cache, pos, np.full(1, ntok), sees, nq, nkv, hd, 0.1, cap)
    check(attend(gpu_ctx, bits, q, cache, pos, counts, sees, nq, nkv, hd, 0.1, cap), want, bound)


def test_attention_masked_scores_above_all_others(gpu_ctx):
    """A token of the block that others do not see scores far above what they do see: it must not take the
    range that their weights are held in."""
    rng = np.random.default_rng(5)
    for bits, hd, nq, nkv, ntok, start in ((8, 64, 2, 1, 20, 100), (4, 128, 8, 2, 64, 30), (8, 128, 4, 4, 140, 0)):
        q, cache, pos, counts, sees, cap = case(rng, bits, 1, ntok, nq, nkv, hd, start, False, False)
        if ntok <= 64:
            sees = np.array([[1 << t for t in range(ntok)]], np.uint64)
        big = slice(start + 1, start + ntok, 2)
        cache[1][0, :, big] = 900.0 if bits == 8 else 0x4461
        want, bound = R.attention(bits, q, cache, pos, np.full(1, ntok), sees, nq, nkv, hd, 0.3, cap)
        check(attend(gpu_ctx, bits, q, cache, pos, counts, sees, nq, nkv, hd, 0.3, cap), want, bound)


def attention_on_gpu(bits, q, cache, pos, counts, sees, nq, nkv, hd, scale, length):
    """block_ref.attention's outputs and bounds for many tokens: a row's KV head at a time in 64 bits on the GPU."""
    import oracle as O
    batch, ntok = q.shape[:2]
    g = nq // nkv
    flat = q.reshape(-1, hd)
    codes = [O.kv_quant_head(x) for x in flat]
    qv = np.stack([c.astype(np.float64) * np.float64(s) for c, s in codes]).reshape(batch, ntok, nkv, g, hd) * float(np.float32(scale))
    out, bound = np.full((batch, ntok, nq, hd), np.nan), np.full((batch, ntok, nq, hd), np.nan)
    for r in range(batch):
        n = int(max(0, min(ntok, counts[r])))
        end = int(max(0, min(length, pos[r] + n)))
        if n == 0:
            continue
        see = torch.from_numpy(R.visible(ntok, int(pos[r]), n, end, None if sees is None else [int(x) for x in sees[r]])[:n]).cuda()
        for h in range(nkv):
            k, v = (dev(B.values(bits, cache[i][r, h, :end], cache[i + 1][r, h, :end])) for i in (0, 2))
            x = dev(qv[r, :n, h]).reshape(n * g, hd)
            parts = (x.view(-1, hd // 64, 64).transpose(0, 1).contiguous() @ k.view(-1, hd // 64, 64).permute(1, 2, 0).contiguous()) if bits == 4 \
                else (x @ k.T.contiguous())[None]
            m = see[:, None].expand(n, g, end).reshape(n * g, end)
            z, size = parts.sum(0).masked_fill(~m, -np.inf), parts.abs().sum(0).masked_fill(~m, 0)
            none = ~m.any(1)
            w = torch.softmax(z, 1).masked_fill(none[:, None], 0)
            o, a = (w @ v).cpu().numpy(), (w @ v.abs()).cpu().numpy()
            rel = (2 * (9 * size.amax(1) + 4) + 2 * (m.sum(1) / 32 + 128)).cpu().numpy()[:, None] * R.U + 2.0 ** -21
            out[r, :n, h * g:(h + 1) * g] = B.unrotate(o).reshape(n, g, hd)
            b = (rel * B.block_sums(a) + 7 * R.U * B.block_sums(np.abs(o))) / 8 + 1e-37
            b[none.cpu().numpy()] = 0
            bound[r, :n, h * g:(h + 1) * g] = b.reshape(n, g, hd)
    return out, bound


# many workgroups of columns (nkv * batch * columns / 128), or a cache of many positions (`room`), of which the rows
# hold few: what is chosen goes by the room
LARGE = [(8, 64, 64, 64, 3, 200, 40, 0, False), (8, 64, 128, 64, 4, 90, 0, 0, True), (8, 128, 96, 48, 5, 130, 70, 0, False),
         (8, 128, 32, 4, 16, 64, 100, 0, True), (4, 64, 66, 33, 6, 150, 30, 0, False), (4, 128, 32, 4, 2, 64, 300, 9000, True),
         (4, 128, 16, 2, 3, 300, 0, 12000, False), (8, 128, 32, 4, 2, 64, 700, 20000, True), (8, 64, 32, 32, 1, 60, 500, 30000, True),
         (8, 128, 8, 2, 2, 40, 900, 6000, False), (4, 64, 9, 3, 3, 50, 40, 50000, True), (8, 64, 12, 4, 1, 1100, 0, 0, False),
         (4, 128, 16, 16, 6, 500, 0, 0, False)]


@pytest.mark.parametrize("bits,hd,nq,nkv,batch,ntok,start,room,with_tree", LARGE)
def test_attention_of_many_columns_and_parts(gpu_ctx, bits, hd, nq, nkv, batch, ntok, start, room, with_tree):
    with_tree = with_tree and ntok <= 64
    print(f"attn_tokens bits={bits} hd={hd} heads={nq}/{nkv} batch={batch} ntok={ntok} start={start} room={room} tree={with_tree}", flush=True)
    rng = np.random.default_rng(hd * ntok + nq)
    q, cache, pos, counts, sees, cap = case(rng, bits, batch, ntok, nq, nkv, hd, start, True, with_tree, spare=3 + room,
                                            first=0 if with_tree else start)
    if with_tree:
        sees[0, ::5] = 0  # (row 0 has nothing in front: these see nothing)
    want, bound = attention_on_gpu(bits, q, cache, pos, counts, sees, nq, nkv, hd, 0.17, cap)
    check(attend(gpu_ctx, bits, q, cache, pos, counts, sees, nq, nkv, hd, 0.17, cap, extra=ntok), want, bound)
    # a NaN and an infinite V scale of one token reach only those that see it
    t = ntok // 3
    r = int(np.argmax(np.minimum(counts, ntok) > t))
    c = [a.copy() for a in cache]
    c[3][r, :, pos[r] + t] = np.nan if bits == 8 else 0x7F80
    got = attend(gpu_ctx, bits, q, c, pos, counts, sees, nq, nkv, hd, 0.17, cap)
    see = R.visible(ntok, int(pos[r]), int(min(counts[r], ntok)), cap, None if sees is None else [int(x) for x in sees[r]])[:, pos[r] + t]
    others = ~np.isnan(bound)
    others[r, see] = False
    assert (np.abs(got - want)[others] <= bound[others]).all()
    assert not np.isfinite(got[r][see & (np.arange(ntok) < counts[r])]).any(-1).all(-1).any()


# items of many columns whose positions workgroups share, each from where the one before stops (few items for two on every CU)
CUT = [(8, 64, 16, 16, 8, 380, 3100, 0, False), (8, 128, 8, 8, 7, 1000, 0, 9000, False), (4, 64, 8, 4, 4, 256, 4100, 0, False),
       (4, 128, 8, 8, 4, 130, 4500, 300, False), (4, 128, 16, 4, 8, 40, 4500, 50, True), (4, 64, 20, 2, 3, 64, 900, 8000, True)]


@pytest.mark.parametrize("bits,hd,nq,nkv,batch,ntok,start,room,with_tree", CUT)
def test_attention_of_items_cut_between_workgroups(gpu_ctx, bits, hd, nq, nkv, batch, ntok, start, room, with_tree):
    print(f"attn_tokens bits={bits} hd={hd} heads={nq}/{nkv} batch={batch} ntok={ntok} start={start} room={room} tree={with_tree}", flush=True)
    rng = np.random.default_rng(hd * ntok + nq)
    q, cache, pos, counts, sees, cap = case(rng, bits, batch, ntok, nq, nkv, hd, start, True, with_tree, spare=3 + room, first=max(0, start - 9))
    counts[1:3] = [0, 1]
    want, bound = attention_on_gpu(bits, q, cache, pos, counts, sees, nq, nkv, hd, 0.17, cap)
    check(attend(gpu_ctx, bits, q, cache, pos, counts, sees, nq, nkv, hd, 0.17, cap), want, bound)


@pytest.mark.parametrize("bits,hd,nq,nkv,batch,ntok,start,room,with_tree", [LARGE[i] for i in (0, 3, 5, 6, 7, 9)])
@pytest.mark.parametrize("kind", ["large", "vscales", "zero", "far"])
def test_attention_of_many_columns_and_values_of_any_size(gpu_ctx, bits, hd, nq, nkv, batch, ntok, start, room, with_tree, kind):
    rng = np.random.default_rng(hd + ntok)
    q, cache, pos, counts, sees, cap = case(rng, bits, batch, ntok, nq, nkv, hd, start, False, with_tree, spare=3 + room)
    end = start + ntok
    shape = cache[1][:, :, :end].shape

    def scales(lo, hi):
        f = np.exp2(rng.uniform(lo, hi, shape)).astype(np.float32)
        return f if bits == 8 else (f.view(np.uint32) >> 16).astype(np.uint16)
    if kind in ("large", "far"):
        cache[1][:, :, :end] = scales(4, 6) if kind == "large" else scales(20, 24)
    elif kind == "vscales":
        cache[3][:, :, :end] = scales(-60, 20)
    else:
        q[:, ::2] = 0.0
    for r in range(batch):
        for a in (cache[1], cache[3]):
            a[r, :, pos[r] + ntok:] = np.nan if bits == 8 else 0x7FC0
    want, bound = attention_on_gpu(bits, q, cache, pos, np.full(batch, ntok), sees, nq, nkv, hd, 0.1, cap)
    check(attend(gpu_ctx, bits, q, cache, pos, counts, sees, nq, nkv, hd, 0.1, cap), want, np.minimum(bound, 1e300))


@pytest.mark.parametrize("bits", [8, 4])
def test_attention_agrees_with_the_one_token_operators(gpu_ctx, bits):
    """A block of one token behind 900 positions is k2t_attn_decode; the largest heads count; rows of their own."""
    rng = np.random.default_rng(bits)
    nq, nkv, hd, n = 16, 4, 128, 900
    cache = B.new_cache(bits, 1, nkv, n + 1, hd, rng)
    q = rng.standard_normal((1, 1, nq, hd)).astype(np.float32)
    got = attend(gpu_ctx, bits, q, cache, np.array([n - 1], np.int32), None, None, nq, nkv, hd, 0.1, n + 1)
    out = torch.zeros(nq, hd, device="cuda")
    t = [dev(a) for a in cache]
    gpu_ctx.attn_decode(bits, dev(q), nq, nkv, hd, *t, n + 1, n, 0.1, out)
    _, bound = R.attention(bits, q, cache, np.array([n - 1]), [1], None, nq, nkv, hd, 0.1, n)
    assert (np.abs(got[0, 0] - out.cpu().numpy()) <= 2 * bound[0, 0]).all()


def test_attention_past_32_bit_offsets(gpu_ctx):
    """A cache of more than 2^32 bytes of codes: its last row and last positions."""
    nkv, hd, cap, batch = 8, 128, 1 << 20, 5
    g = torch.Generator(device="cuda").manual_seed(2)
    k, v = (torch.zeros(batch * nkv * cap, hd, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.full((batch * nkv * cap,), 0.01, device="cuda") for _ in range(2))
    start, ntok, nq = cap - 30, 20, 16
    small = []
    for a in (k, v):
        tail = torch.randint(-127, 128, (batch, nkv, 40, hd), generator=g, device="cuda", dtype=torch.int8)
        a.view(batch, nkv, cap, hd)[:, :, -40:] = tail
        small.append(tail)
    # positions before the last forty score 0 and add nothing but to the sum: few enough not to matter to the check's bound
    kv = k2t.KVRows(k, ks, v, vs, cap=cap)
    q = 4 * torch.randn(batch * ntok, nq * hd, generator=g, device="cuda")
    out = torch.zeros(batch * ntok, nq * hd, device="cuda")
    ws = workspace(gpu_ctx.attn_tokens_workspace(batch, ntok, nq, nkv, hd, cap))
    gpu_ctx.attn_tokens(8, q, nq * hd, batch, ntok, nq, nkv, hd, ints([start] * batch), kv, 1.0, out, ws)
    gpu_ctx.sync()
    got = out.cpu().numpy().reshape(batch, ntok, nq, hd)
    import oracle as O
    for r, t, h in ((batch - 1, ntok - 1, nq - 1), (0, 0, 0), (batch - 1, 0, 3)):
        code, qs = O.kv_quant_head(q.view(batch, ntok, nq, hd)[r, t, h].cpu().numpy())
        seen = start + t + 1 - (cap - 40)
        kk, vv = (x[r, h // 2, :seen].cpu().numpy().astype(np.float64) * float(np.float32(0.01)) for x in small)
        z = kk @ (code * np.float64(qs))
        m = max(z.max(), 0.0)
        w = np.exp(z - m)
        total = w.sum() + (cap - 40) * np.exp(-m)
        o = (w / total) @ vv
        S = max(np.abs(z).max(), m)
        rel = (2 * (9 * S + 4) + 2 * (cap / 32 + 128)) * R.U + 2.0 ** -21
        bound = (rel * B.block_sums((w / total) @ np.abs(vv)) + 7 * R.U * B.block_sums(np.abs(o))) / 8 + 1e-37
        assert (np.abs(got[r, t, h] - B.unrotate(o)) <= bound).all(), (r, t, h)


# ---------------------------------------------------------------- logits
def adjust(ctx, x, vocab, rules, in_place, shift=0):
    rows, stride = x.shape
    buf = torch.full((rows * stride + 8,), 3.25, device="cuda")
    at = buf[shift:shift + rows * stride].view(rows, stride)
    at.copy_(dev(x))
    d = {n: dev(a) for n, a in rules.items()}
    out = at if in_place else torch.full((rows, stride), 3.25, device="cuda")
    ctx.logits_adjust(at, vocab, stride, rows, k2t.LogitsRules(**d), out, stride)
    ctx.sync()
    if not in_place:
        assert np.array_equal(at.cpu().numpy().view(np.uint32), x.view(np.uint32))
        assert (out[:, vocab:] == 3.25).all()
    assert (buf[:shift] == 3.25).all() and (buf[shift + rows * stride:] == 3.25).all()
    return out.cpu().numpy()


def rules_for(rng, rows, vocab, history, bias, masked):
    d = {}
    if history:
        h = (vocab * rng.random((rows, history)) ** 3).astype(np.int32)
        h[rng.random(h.shape) < 0.05] = -1
        h[rng.random(h.shape) < 0.05] = vocab
        d.update(history=h, history_len=rng.integers(-1, history + 3, rows).astype(np.int32),
                 prompt_len=rng.integers(-2, history + 2, rows).astype(np.int32),
                 repeat=rng.uniform(0.8, 1.5, rows).astype(np.float32), presence=rng.uniform(-1, 1, rows).astype(np.float32),
                 frequency=rng.uniform(0, 1, rows).astype(np.float32))
        d["history_len"][0] = history
    if bias:
        t = rng.integers(-2, vocab + 2, (rows, bias)).astype(np.int32)
        t[:, bias // 2:] = t[:, :bias - bias // 2]  # twice the same tokens
        d.update(bias_tokens=t, bias=(7 * rng.standard_normal((rows, bias))).astype(np.float32),
                 bias_len=rng.integers(-1, bias + 2, rows).astype(np.int32))
        d["bias_len"][-1] = bias
        d["bias"][-1, 0] = -np.inf
    if masked:
        d.update(mask=rng.integers(-2 ** 31, 2 ** 31, (3, (vocab + 31) // 32 + 1)).astype(np.int32),
                 mask_row=rng.integers(-1, 4, rows).astype(np.int32))
    return d


@pytest.mark.parametrize("rows,vocab,history,bias,masked", [
    (1, 1, 1, 1, True), (3, 31, 5, 3, True), (2, 4096, 300, 0, False), (5, 4097, 70, 40, True), (1, 8191, 3000, 0, True), (4, 9000, 0, 300, False),
    (2, 50257, 1000, 64, True), (3, 700, 0, 0, True), (2, 515, 0, 0, False), (1, 20000, 40, 4096, False)])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("pad", [0, 3])
def test_logits_adjust(gpu_ctx, rows, vocab, history, bias, masked, in_place, pad):
    print(f"logits rows={rows} vocab={vocab} history={history} bias={bias} masked={masked} in_place={in_place}", flush=True)
    rng = np.random.default_rng(rows * vocab + history)
    x = (4 * rng.standard_normal((rows, vocab + pad))).astype(np.float32)
    rules = rules_for(rng, rows, vocab, history, bias, masked)
    want = R.logits(x, vocab, rules)
    got = adjust(gpu_ctx, x, vocab, rules, in_place, shift=pad % 4)
    assert np.array_equal(got[:, :vocab], want[:, :vocab])
    if in_place:
        assert np.array_equal(got, want)
    # each list alone
    for names in (("history", "repeat"), ("history", "presence"), ("history", "history_len", "frequency"), ("bias_tokens", "bias"), ("mask", "mask_row")):
        part = {n: rules[n] for n in names if n in rules}
        if len(part) == len(names):
            assert np.array_equal(adjust(gpu_ctx, x, vocab, part, in_place)[:, :vocab], R.logits(x, vocab, part)[:, :vocab])


def test_logits_of_odd_values(gpu_ctx):
    """NaN keep their bits where nothing applies, infinities follow the formula, -inf masks win, sums overflow."""
    x = np.array([[np.nan, np.inf, -np.inf, 0.0, -0.0, 3e38, -3e38, 1e-40, np.nan, np.inf]], np.float32)
    x.view(np.uint32)[0, 0] = 0x7FC12345
    rules = dict(history=np.arange(1, 8, dtype=np.int32)[None], repeat=np.array([2.0], np.float32), presence=np.array([1.0], np.float32),
                 frequency=np.array([0.5], np.float32), bias_tokens=np.array([[6, 6, 5, 8]], np.int32),
                 bias=np.array([[-3e38, -3e38, 3e38, 1.0]], np.float32), mask=np.array([[0x1FF]], np.int32))
    with np.errstate(over="ignore"):
        want = R.logits(x, 10, rules)
    for in_place in (False, True):
        got = adjust(gpu_ctx, x, 10, rules, in_place)
        assert np.array_equal(got, want, equal_nan=True) and got.view(np.uint32)[0, 0] == 0x7FC12345
        assert got[0, 9] == -np.inf and np.isnan(got[0, 8]) and got[0, 6] == -np.inf


def test_logits_of_the_longest_lists(gpu_ctx):
    """2^20 tokens of history, one of them half of the time; 4096 biases of one token, added in the list's order."""
    rng = np.random.default_rng(1)
    vocab = 151936
    x = rng.standard_normal((2, vocab)).astype(np.float32)
    h = rng.integers(0, vocab, (2, 1 << 20)).astype(np.int32)
    h[:, ::2] = 77
    rules = dict(history=h, frequency=np.array([0.01, 0.25], np.float32), repeat=np.array([1.1, 1.3], np.float32),
                 bias_tokens=np.full((2, 4096), 5, np.int32), bias=(rng.standard_normal((2, 4096)) * 1000).astype(np.float32))
    assert np.array_equal(adjust(gpu_ctx, x, vocab, rules, False), R.logits(x, vocab, rules))


# ---------------------------------------------------------------- keep
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("layers,rows,nkv,cap,n_keep", [(1, 1, 1, 1, 1), (2, 3, 2, 40, 9), (1, 2, 3, 700, 300), (3, 1, 1, 5000, 4000), (1, 4, 1, 130, 129), (9, 30, 1, 700, 300)])
def test_keep(gpu_ctx, bits, hd, layers, rows, nkv, cap, n_keep):
    print(f"kv_keep bits={bits} hd={hd} layers={layers} rows={rows} nkv={nkv} cap={cap} n_keep={n_keep}", flush=True)
    rng = np.random.default_rng(cap + n_keep)
    cache = [a.reshape(layers, rows, *a.shape[1:]) for a in B.new_cache(bits, layers * rows, nkv, cap, hd, rng)]
    for kind in ("sorted", "odd", "shift"):
        pos = rng.integers(0, max(1, cap - n_keep), rows).astype(np.int32)
        counts = rng.integers(0, n_keep + 2, rows).astype(np.int32)
        counts[0] = n_keep
        if kind == "sorted":  # an eviction
            lists = np.stack([np.sort(rng.permutation(cap)[:n_keep]) for _ in range(rows)]).astype(np.int32)
            pos[:] = 0
        elif kind == "shift":  # everything moves by the same distance
            lists = np.tile(np.arange(n_keep, dtype=np.int32) + min(17, cap - 1), (rows, 1))
        else:  # entries below their place, twice the same, outside the cache, negative; rows that begin outside it
            lists = rng.integers(-2, cap + 3, (rows, n_keep)).astype(np.int32)
            pos[-1] = -3
        t, kv = rows_of(cache, cap, length=0)
        wide = np.full((rows, n_keep + 2), -9, np.int32)
        wide[:, :n_keep] = lists
        gpu_ctx.kv_keep(bits, kv, dev(pos), dev(wide), n_keep + 2, dev(counts), n_keep, layers, rows, nkv, hd)
        gpu_ctx.sync()
        for g, w in zip(t, R.keep(cache, pos, lists, counts, n_keep)):
            assert np.array_equal(host(g, w), w), kind
        t, kv = rows_of(cache, cap)
        gpu_ctx.kv_keep(bits, kv, dev(pos), dev(lists), n_keep, None, n_keep, layers, rows, nkv, hd)
        gpu_ctx.sync()
        for g, w in zip(t, R.keep(cache, pos, lists, None, n_keep)):
            assert np.array_equal(host(g, w), w), kind


def test_keep_past_32_bit_offsets(gpu_ctx):
    """A cache of more than 2^32 bytes of codes: the last row's last positions."""
    nkv, hd, cap = 1, 128, 1 << 24
    layers = 3
    k, v = (torch.zeros(layers * cap, hd, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(layers * cap, device="cuda") for _ in range(2))
    ends = (torch.arange(layers, device="cuda")[:, None] + 1) * cap - 100 + torch.arange(100, device="cuda")
    tail = torch.randint(-127, 128, (layers, 100, hd), device="cuda", dtype=torch.int8)
    k[ends], v[ends] = tail, tail.flip(-1)
    ks[ends], vs[ends] = tail[..., 0].float(), tail[..., 1].float()
    kv = k2t.KVRows(k, ks, v, vs, cap=cap)
    lists = torch.sort(torch.randperm(100)[:60]).values.int()[None].contiguous().cuda()
    gpu_ctx.kv_keep(8, kv, ints([cap - 100]), lists, 60, None, 60, layers, 1, nkv, hd)
    gpu_ctx.sync()
    want = tail.clone()
    want[:, :60] = tail[:, lists[0].long()]
    assert torch.equal(k[ends], want) and torch.equal(ks[ends], want[..., 0].float()) and torch.equal(vs[ends], want[..., 1].float())
    assert torch.equal(v[ends], want.flip(-1))


# ---------------------------------------------------------------- a run of them
class Sequences:
    """A batch of sequences over one layer's cache: fixed projections of token embeddings stand for a model."""

    def __init__(self, ctx, bits, rows, nq, nkv, hd, cap, vocab, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.ctx, self.bits, self.rows, self.nq, self.nkv, self.hd, self.cap, self.vocab = ctx, bits, rows, nq, nkv, hd, cap, vocab
        self.width = (nq + 2 * nkv) * hd
        self.embed = torch.randn(vocab, self.width, generator=g, device="cuda")
        self.head = torch.randn(nq * hd, vocab, generator=g, device="cuda") / (nq * hd) ** 0.5
        codes = torch.int8 if bits == 8 else torch.uint8
        n, w = (rows, nkv, cap), hd if bits == 8 else hd // 2
        self.t = [torch.zeros(*n, w, dtype=codes, device="cuda"), torch.zeros(*n, *(() if bits == 8 else (hd // 64,)),
                                                                              dtype=torch.float32 if bits == 8 else torch.bfloat16, device="cuda")]
        self.t += [a.clone() for a in self.t]
        self.kv = k2t.KVRows(*self.t, cap=cap)
        self.plan = k2t.RopePlan(k2t.ROPE_HALF, hd, 10000.0)

    def step(self, tokens, pos, counts=None, sees=None, depth=None):
        """Tokens [rows][ntok] at pos: the attention's logits [rows * ntok][vocab]."""
        ntok, at = tokens.shape[1], lambda x, off: x.data_ptr() + 4 * off
        x = self.embed[tokens.reshape(-1).long()].contiguous()
        nq, nkv, hd = self.nq, self.nkv, self.hd
        self.ctx.rope(x, self.width, self.rows, ntok, nq + nkv, hd, pos, self.plan, x, self.width, depth=depth, counts=counts)
        self.ctx.kv_append(self.bits, at(x, nq * hd), at(x, (nq + nkv) * hd), self.width, self.rows, ntok, nkv, hd, pos, self.kv, counts=counts)
        out = torch.zeros(self.rows * ntok, nq * hd, device="cuda")
        ws = workspace(self.ctx.attn_tokens_workspace(self.rows, ntok, nq, nkv, hd, self.cap))
        self.ctx.attn_tokens(self.bits, x, self.width, self.rows, ntok, nq, nkv, hd, pos, self.kv, hd ** -0.5, out, ws, counts=counts, sees=sees)
        self.ctx.sync()
        return (out.double() @ self.head.double()).float()

    def pick(self, logits, history, lens):
        """The best token of every row after a repetition penalty, by k2t_beam_select of one beam."""
        rows = logits.shape[0]
        rules = k2t.LogitsRules(history=history, history_len=lens, repeat=torch.full((rows,), 1.2, device="cuda"))
        self.ctx.logits_adjust(logits, self.vocab, self.vocab, rows, rules, logits, self.vocab)
        o = [torch.zeros(rows, 1, dtype=d, device="cuda") for d in (torch.float32, torch.int32, torch.int32)]
        ws = workspace(self.ctx.beam_select_workspace(rows, 1, self.vocab, 1))
        self.ctx.beam_select(logits, self.vocab, self.vocab, torch.zeros(rows, device="cuda"), None, rows, 1, 1, -1, *o, None, ws)
        self.ctx.sync()
        return o[1].view(-1)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("nq,nkv,hd", [(4, 2, 64), (8, 1, 128)])
def test_drafted_trees_decode_what_single_tokens_decode(gpu_ctx, bits, nq, nkv, hd):
    """Prompts of different lengths, then rounds that check a drafted tree each and keep the path that the picks
    agree with: the same tokens and the same cache as one token at a time. The drafts hold the right
    continuation on scattered branches, now and then with a wrong turn."""
    rows, prompt, cap, vocab, total = 3, 40, 128, 600, 24
    rng = np.random.default_rng(bits + hd)
    tokens = torch.from_numpy(rng.integers(0, vocab, (rows, prompt)).astype(np.int32)).cuda()
    lens = ints([40, 23, 31])

    def start():
        s = Sequences(gpu_ctx, bits, rows, nq, nkv, hd, cap, vocab)
        logits = s.step(tokens, ints([0] * rows), counts=lens).view(rows, prompt, vocab)
        return s, logits[torch.arange(rows), lens.long() - 1].contiguous()

    # one token at a time
    s, logits = start()
    seqs = [tokens[r, :lens[r]].tolist() for r in range(rows)]
    hist = torch.zeros(rows, cap, dtype=torch.int32, device="cuda")
    pos = lens.clone()

    def history(seqs):
        for r, q in enumerate(seqs):
            hist[r, :len(q)] = torch.tensor(q, dtype=torch.int32)
        return hist, ints([len(q) for q in seqs])

    for _ in range(total + 8):
        nxt = s.pick(logits, *history(seqs))
        for r in range(rows):
            seqs[r].append(int(nxt[r]))
        logits = s.step(nxt.view(rows, 1).contiguous(), pos)
        pos = pos + 1
    single = s
    # drafted trees
    s, logits = start()
    got = [tokens[r, :lens[r]].tolist() for r in range(rows)]
    pos = lens.clone()
    nxt = s.pick(logits, *history(got))
    while min(len(g) - int(n) for g, n in zip(got, lens)) < total:
        ntok = int(rng.integers(2, 12))
        draft, parent = np.zeros((rows, ntok), np.int32), np.full((rows, ntok), -1)
        for r in range(rows):
            draft[r, 0] = int(nxt[r])
            tip = 0
            for t in range(1, ntok):
                right = seqs[r][len(got[r]) + 1 + sum(1 for _ in path(parent[r], tip))] if len(got[r]) + ntok + 2 < len(seqs[r]) else 0
                if rng.random() < 0.6:  # the right continuation of the longest right path
                    draft[r, t], parent[r, t], tip = right, tip, t
                else:
                    draft[r, t], parent[r, t] = rng.integers(0, vocab), rng.integers(0, t)
        sees, depth = np.zeros((rows, ntok), np.int64), np.zeros((rows, ntok), np.int32)
        for r in range(rows):
            for t in range(ntok):
                up = [t] + list(path(parent[r], t))
                sees[r, t], depth[r, t] = sum(1 << u for u in up), len(up) - 1
        counts = ints(rng.integers((ntok + 1) // 2, ntok + 1, rows).tolist())
        logits = s.step(dev(draft), pos, counts=counts, sees=dev(sees), depth=dev(depth))
        # every token's history: its row's, then its path
        flat, n = torch.zeros(rows * ntok, cap, dtype=torch.int32, device="cuda"), []
        for r in range(rows):
            for t in range(ntok):
                h = got[r] + [int(draft[r, u]) for u in reversed([t] + list(path(parent[r], t)))]
                flat[r * ntok + t, :len(h)] = torch.tensor(h, dtype=torch.int32)
                n.append(len(h))
        picks = s.pick(logits, flat, ints(n)).view(rows, ntok).cpu().numpy()
        lists, kept = np.zeros((rows, ntok), np.int32), []
        for r in range(rows):
            at, line = 0, [0]
            while True:
                child = [t for t in range(1, int(counts[r])) if parent[r, t] == at and draft[r, t] == picks[r, at]]
                if not child:
                    break
                at = child[0]
                line.append(at)
            lists[r, :len(line)] = line
            kept.append(len(line))
            got[r] += [int(draft[r, t]) for t in line]
            nxt[r] = int(picks[r, at])
        gpu_ctx.kv_keep(bits, s.kv, pos, dev(lists), ntok, ints(kept), ntok, 1, rows, nkv, hd)
        pos = pos + ints(kept)
    gpu_ctx.sync()
    for r in range(rows):
        n = int(lens[r]) + total
        assert got[r][:n] == seqs[r][:n]
        for a, b in zip(s.t, single.t):  # the cache holds the same bytes: rope at its depth, append, keep
            assert torch.equal(a[r, :, :n].view(torch.uint8), b[r, :, :n].view(torch.uint8))


def path(parent, t):
    """The ancestors of t, nearest first."""
    while parent[t] >= 0:
        t = parent[t]
        yield t


def test_calls_in_a_graph_follow_what_is_on_the_device():
    """All four captured together on another stream; the replays read positions, counts, masks, histories and lists as they are then."""
    stream = torch.cuda.Stream()
    ctx = k2t.Ctx(0, stream)
    rows, ntok, nq, nkv, hd, cap, vocab = 2, 6, 8, 2, 64, 600, 5000
    g = torch.Generator(device="cuda").manual_seed(4)
    new = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    x0, logits0 = new(rows * ntok, nq * hd), new(rows, vocab)
    cache0 = [torch.randint(-127, 128, (rows, nkv, cap, hd), generator=g, device="cuda", dtype=torch.int8), 0.02 * torch.ones(rows, nkv, cap, device="cuda")]
    cache0 += [a.clone() for a in cache0]
    plan = k2t.RopePlan(k2t.ROPE_HALF, hd, 1e4)
    pos, counts, sees = ints([500, 40]), ints([6, 3]), torch.full((rows, ntok), 63, dtype=torch.int64, device="cuda")
    hist, lists = torch.randint(0, vocab, (rows, 50), generator=g, device="cuda", dtype=torch.int32), ints([[0, 2, 5], [0, 1, 4]])
    rules = k2t.LogitsRules(history=hist, frequency=torch.ones(rows, device="cuda"))
    x, out, logits = (torch.zeros_like(a) for a in (x0, x0, logits0))
    cache = [a.clone() for a in cache0]
    ws = workspace(ctx.attn_tokens_workspace(rows, ntok, nq, nkv, hd, cap))

    def calls(c, x, out, logits, cache, ws):
        kv = k2t.KVRows(*cache, cap=cap)
        c.rope(x0, nq * hd, rows, ntok, nq, hd, pos, plan, x, nq * hd, counts=counts)
        c.attn_tokens(8, x, nq * hd, rows, ntok, nq, nkv, hd, pos, kv, 0.125, out, ws, counts=counts, sees=sees)
        c.logits_adjust(logits0, vocab, vocab, rows, rules, logits, vocab)
        c.kv_keep(8, kv, pos, lists, 3, None, 3, 1, rows, nkv, hd)

    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        calls(ctx, x, out, logits, cache, ws)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            calls(ctx, x, out, logits, cache, ws)
        eager = k2t.Ctx(0, stream)
        for i in range(4):
            pos.copy_(ints([[500, 40], [3, 590], [0, 1], [594, 77]][i]))
            counts.copy_(ints([[6, 3], [5, 6], [1, 0], [6, 6]][i]))
            sees.fill_([63, 21, 0, 33][i])
            hist.add_(1).remainder_(vocab)
            lists.copy_(ints([[[0, 2, 5], [0, 1, 4]], [[1, 2, 3], [5, 5, 5]], [[0, 0, 0], [2, 3, 4]], [[3, 4, 5], [0, 5, 9]]][i]))
            for a, b in zip(cache, cache0):
                a.copy_(b)
            x.zero_(), out.zero_(), logits.zero_()
            stream.synchronize()
            graph.replay()
            stream.synchronize()
            want = [torch.zeros_like(a) for a in (x, out, logits)] + [a.clone() for a in cache0]
            calls(eager, *want[:3], want[3:], workspace(ws.numel()))
            stream.synchronize()
            for a, b in zip([x, out, logits, *cache], want):
                assert torch.equal(a, b), i
        eager.close()
    ctx.close()


# ---------------------------------------------------------------- the largest calls, and calls beside each other
def test_the_most_rows_of_blocks(gpu_ctx):
    """65535 rows of one token in one call of each kind: what a call of few rows does to each of them."""
    rows, few, hd, cap = 65535, 7, 64, 3
    g = torch.Generator(device="cuda").manual_seed(3)
    many = torch.arange(rows, device="cuda") % few
    x = torch.randn(few, hd, generator=g, device="cuda")
    cache = [torch.randint(-127, 128, (few, 1, cap, hd), generator=g, device="cuda", dtype=torch.int8),
             torch.rand(few, 1, cap, generator=g, device="cuda")]
    cache += [a.flip(0).contiguous() for a in cache]
    pos, lists = ints([2, 0, 1, 2, 2, 1, 0]), ints([[i % 3, 2] for i in range(few)])
    rules = dict(history=ints([[i, i, 4 - i % 5] for i in range(few)]), frequency=torch.rand(few, generator=g, device="cuda"))
    logits = torch.randn(few, 5, generator=g, device="cuda")
    plan = k2t.RopePlan(k2t.ROPE_INTERLEAVED, 30, 1e4)

    def calls(n, x, cache, pos, lists, rules, logits):
        out, rot, adj = torch.zeros(n, hd, device="cuda"), torch.zeros(n, hd, device="cuda"), torch.zeros(n, 5, device="cuda")
        kv = k2t.KVRows(*cache, cap=cap)
        ws = workspace(gpu_ctx.attn_tokens_workspace(n, 1, 1, 1, hd, cap))
        gpu_ctx.attn_tokens(8, x, hd, n, 1, 1, 1, hd, pos, kv, 0.1, out, ws)
        gpu_ctx.rope(x, hd, n, 1, 1, hd, pos, plan, rot, hd)
        gpu_ctx.logits_adjust(logits, 5, 5, n, k2t.LogitsRules(**rules), adj, 5)
        gpu_ctx.kv_keep(8, kv, torch.zeros_like(pos), lists, 2, None, 2, 1, n, 1, hd)
        gpu_ctx.sync()
        return [out, rot, adj, *cache]

    take = lambda t: t[many].contiguous()  # noqa: E731
    got = calls(rows, take(x), [take(a) for a in cache], take(pos), take(lists), {n: take(a) for n, a in rules.items()}, take(logits))
    want = calls(few, x, cache, pos, lists, rules, logits)
    assert want[0].abs().min(1).values.min() > 0 and not torch.equal(want[1], x) and not torch.equal(want[2], logits)
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8), take(b).view(torch.uint8))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("nq,nkv,ntok", [(1024, 1, 2), (1024, 1024, 3), (1024, 32, 5)])
def test_attention_of_the_most_heads(gpu_ctx, bits, nq, nkv, ntok):
    print(f"attn_tokens bits={bits} heads={nq}/{nkv} ntok={ntok}", flush=True)
    rng = np.random.default_rng(nkv)
    q, cache, pos, counts, sees, cap = case(rng, bits, 2, ntok, nq, nkv, 64, 37, True, True)
    got = attend(gpu_ctx, bits, q, cache, pos, counts, sees, nq, nkv, 64, 0.17, cap)
    check(got, *R.attention(bits, q, cache, pos, counts, sees, nq, nkv, 64, 0.17, cap))


def test_strides_past_32_bits(gpu_ctx):
    """Rows 2^31 floats apart, and more than 2^32 bytes."""
    stride, hd, vocab = (1 << 31) + 64, 64, 6
    buf = torch.empty(2 * stride, device="cuda")
    x = torch.randn(3, hd, device="cuda")
    at = [buf[i * stride:i * stride + hd] for i in range(2)] + [buf[-hd:]]
    plan = k2t.RopePlan(k2t.ROPE_HALF, hd, 1e4)
    want, out = torch.zeros(2, hd, device="cuda"), torch.zeros(2, hd, device="cuda")
    for i in range(2):
        at[i].copy_(x[i])
    gpu_ctx.rope(x, hd, 1, 2, 1, hd, ints([9]), plan, want, hd)
    gpu_ctx.rope(buf, stride, 1, 2, 1, hd, ints([9]), plan, out, hd)
    gpu_ctx.rope(buf, stride, 1, 2, 1, hd, ints([9]), plan, buf, stride)
    gpu_ctx.sync()
    assert torch.equal(out, want) and torch.equal(torch.stack(at[:2]), want)
    rules = k2t.LogitsRules(history=ints([[0, 2], [5, 9]]), repeat=torch.tensor([2.0, 4.0], device="cuda"))
    gpu_ctx.logits_adjust(buf, vocab, stride, 2, rules, buf, stride)
    gpu_ctx.sync()
    for i, tokens in enumerate(([0, 2], [5])):
        r = 2.0 * (i + 1)
        for t in tokens:
            want[i, t] = want[i, t] / r if want[i, t] > 0 else want[i, t] * r
    assert torch.equal(torch.stack(at[:2]), want)


@pytest.mark.parametrize("bits,hd,nq,nkv,ntok,start", [(8, 64, 9, 3, 10, 300), (8, 128, 32, 4, 300, 2000), (4, 128, 16, 4, 600, 900)])
def test_contexts_on_two_streams_do_not_meet(bits, hd, nq, nkv, ntok, start):
    """Two contexts' calls under way at once, each with a workspace and buffers of its own: the results of each alone."""
    rng = np.random.default_rng(ntok)
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [k2t.Ctx(0, s) for s in streams]
    cap = start + ntok
    runs = []
    for c in ctxs:
        t, kv = rows_of(B.new_cache(bits, 1, nkv, cap, hd, rng), cap)
        q = torch.from_numpy(rng.standard_normal((ntok, nq * hd)).astype(np.float32)).cuda()
        runs.append((c, t, kv, q, ints([start]), workspace(c.attn_tokens_workspace(1, ntok, nq, nkv, hd, cap)),
                     [torch.zeros(ntok, nq * hd, device="cuda") for _ in range(6)]))
    torch.cuda.synchronize()

    def go(run, i):
        c, t, kv, q, pos, ws, out = run
        c.attn_tokens(bits, q, nq * hd, 1, ntok, nq, nkv, hd, pos, kv, 0.125, out[i], ws)

    for run in runs:
        go(run, 0)
        run[0].sync()
    for i in range(1, 6):
        for run in runs:
            go(run, i)
    for run, c in zip(runs, ctxs):
        c.sync()
        assert run[6][0].abs().sum() > 0
        for o in run[6][1:]:
            assert torch.equal(o, run[6][0])
    for c in ctxs:
        c.close()


# ---------------------------------------------------------------- scores past whole numbers, with V scales apart
def exponents(bits, rng, shape, lo, hi):
    """Scales 2^lo .. 2^hi of the cache's type."""
    f = np.exp2(rng.uniform(lo, hi, shape)).astype(np.float32)
    return f if bits == 8 else (f.view(np.uint32) >> 16).astype(np.uint16)


def check_best(got, bits, q, cache, pos, counts, sees, nq, nkv, hd, scale, length):
    """Where a token's best visible position leads by more than rounding leaves open, and by enough for the others to
    weigh nothing next to their V scales, its output is that position's V.  A score is off by 5 roundings of the largest.
    Returns the share of (token, head) that are told apart."""
    import oracle as O
    batch, ntok = q.shape[:2]
    g, told, every = nq // nkv, 0, 0
    for r in range(batch):
        n = int(max(0, min(ntok, counts[r])))
        end = int(max(0, min(length, pos[r] + n)))
        if n == 0 or end == 0:
            continue
        see = R.visible(ntok, int(pos[r]), n, end, None if sees is None else [int(x) for x in sees[r]])[:n]
        see_h, rows = np.repeat(see, g, 0), np.repeat(see.any(1), g)
        for h in range(nkv):
            k, v = (B.values(bits, cache[i][r, h, :end], cache[i + 1][r, h, :end]) for i in (0, 2))
            vs = cache[3][r, h, :end] if bits == 8 else B.bf16(cache[3][r, h, :end])
            lv = np.log2(vs.astype(np.float64)).reshape(end, -1)
            heads = q[r, :n, h * g:(h + 1) * g].reshape(n * g, hd)
            x = np.stack([c.astype(np.float64) * np.float64(s) for c, s in (O.kv_quant_head(a) for a in heads)])
            z = np.where(see_h, (x @ k.T) * float(np.float32(scale)), -np.inf)
            best = z.argmax(1)
            size = np.abs(np.where(see_h, z, 0)).max(1, keepdims=True)
            apart = (lv[None] - lv[best][:, None]).max(-1)
            gap = z[np.arange(n * g), best][:, None] - z - 10 * R.U * size - np.log(2) * (45 + np.maximum(apart, 0))
            gap[np.arange(n * g), best] = np.inf
            ok = (gap.min(1) >= 0) & rows
            out = got[r, :n, h * g:(h + 1) * g].reshape(n * g, hd)
            assert np.isfinite(out).all()
            want = B.unrotate(v[best])
            # pieces of 2^-21, a sum of one term, the rotation's 8 roundings, all others together 2^-30
            bound = (2.0 ** -21 + 8 * R.U + 2.0 ** -30) * B.block_sums(np.abs(v[best])) / 8
            off = np.abs(out - want) > bound
            assert not off[ok].any(), (r, h, np.argwhere(off & ok[:, None])[:4], out[ok][off[ok]][:4], want[ok][off[ok]][:4])
            told += int(ok.sum())
            every += int(rows.sum())
    return told / max(1, every)


# few columns of one tile and of two, in one part and in several; many columns, whole and cut; one token
FAR = [(3, 9, 3, 5, 300, 0, True), (1, 8, 1, 3, 700, 0, False), (2, 4, 2, 64, 100, 0, True), (1, 64, 8, 40, 30, 0, False), (2, 32, 4, 64, 700, 20000, True),
       (3, 96, 48, 130, 70, 0, False), (3, 16, 2, 300, 10, 12000, False), (7, 1, 1, 1, 200, 0, False)]


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("batch,nq,nkv,ntok,start,room,with_tree", FAR)
@pytest.mark.parametrize("size", [2.9e6, 1.1e7, 3e7, 1e9, 1e13])
def test_attention_of_far_scores_and_scales_far_apart(gpu_ctx, bits, hd, batch, nq, nkv, ntok, start, room, with_tree, size):
    """Scores of 2.9e6 (2^22 powers of two) to 1e13 and V scales 2^-30 .. 2^30: a large scale of small weight, or of a
    position that the token does not see, takes nothing from the best position's V."""
    print(f"far bits={bits} hd={hd} heads={nq}/{nkv} batch={batch} ntok={ntok} start={start} room={room} size={size}", flush=True)
    rng = np.random.default_rng(hd + ntok + nq)
    q, cache, pos, counts, sees, cap = case(rng, bits, batch, ntok, nq, nkv, hd, start, False, with_tree, spare=3 + room)
    shape = cache[3].shape
    cache[3][:] = exponents(bits, rng, shape, -30, 30)
    for r in range(batch):  # what lies behind a row's block: any scale
        cache[1][r, :, pos[r] + ntok:] = exponents(bits, rng, cache[1][r, :, pos[r] + ntok:].shape, -60, 60)
        cache[3][r, :, pos[r] + ntok:] = exponents(bits, rng, cache[3][r, :, pos[r] + ntok:].shape, 60, 100)
    # |q . k| of these is about sqrt(hd) * 2 at one standard deviation
    scale = np.float32(size / (4 * 2 * hd ** 0.5))
    got = attend(gpu_ctx, bits, q, cache, pos, counts, sees, nq, nkv, hd, float(scale), cap)
    assert check_best(got, bits, q, cache, pos, np.full(batch, ntok), sees, nq, nkv, hd, scale, cap) >= 0.6


@pytest.mark.parametrize("bits,hd", [(8, 64), (8, 128), (4, 64), (4, 128)])
@pytest.mark.parametrize("nq,nkv,ntok,start,with_tree", [(4, 2, 12, 60, True), (8, 1, 40, 20, False), (8, 8, 200, 0, False), (48, 1, 300, 100, False)])
def test_attention_of_a_far_query_leaves_the_others_bits(gpu_ctx, bits, hd, nq, nkv, ntok, start, with_tree):
    """Heads whose scores are far, between heads whose scores are not: the others' outputs keep their bits."""
    rng = np.random.default_rng(hd + ntok)
    q, cache, pos, counts, sees, cap = case(rng, bits, 2, ntok, nq, nkv, hd, start, False, with_tree)
    cache[3][:] = exponents(bits, rng, cache[3].shape, -12, 12)
    for r in range(2):
        cache[3][r, :, pos[r] + ntok:] = np.nan if bits == 8 else 0x7FC0
    far = rng.random((2, ntok, nq)) < 0.2
    both = np.where(far[..., None], np.float32(2.0 ** 26) * q, q)
    plain = attend(gpu_ctx, bits, q, cache, pos, counts, sees, nq, nkv, hd, 0.17, cap)
    got = attend(gpu_ctx, bits, both, cache, pos, counts, sees, nq, nkv, hd, 0.17, cap)
    assert got[~far].tobytes() == plain[~far].tobytes()
    assert np.isfinite(got).all()


@pytest.mark.parametrize("nq,nkv,ntok,start", [(2, 1, 3, 40), (8, 2, 40, 300), (32, 8, 200, 100), (64, 32, 130, 0)])
@pytest.mark.parametrize("first,second", [(2.0 ** 20, 0.0), (2.0 ** 60, 0.0), (0.0, 2.0 ** 60), (2.0 ** 25, 2.0 ** -80), (0.0, 0.0)])
def test_attention_of_nf4_blocks_of_scales_far_apart(gpu_ctx, nq, nkv, ntok, start, first, second):
    """The two V blocks of a head of 128: one of zeros, or one 2^105 times the other."""
    rng = np.random.default_rng(ntok)
    q, cache, pos, counts, sees, cap = case(rng, 4, 2, ntok, nq, nkv, 128, start, False, False)
    for b, size in ((0, first), (1, second)):
        f = (rng.uniform(1, 2, cache[3].shape[:3]) * size).astype(np.float32)
        cache[3][..., b] = (f.view(np.uint32) >> 16).astype(np.uint16)
    want, bound = attention_on_gpu(4, q, cache, pos, np.full(2, ntok), sees, nq, nkv, 128, 0.17, cap)
    check(attend(gpu_ctx, 4, q, cache, pos, counts, sees, nq, nkv, 128, 0.17, cap), want, bound)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd,nq,nkv,ntok,start", [(64, 2, 2, 12, 50), (128, 8, 2, 40, 200), (128, 16, 2, 64, 1500), (64, 40, 8, 150, 0)])
def test_attention_beside_the_largest_scales(gpu_ctx, bits, hd, nq, nkv, ntok, start):
    """A token's V scale, or K scale, of up to the largest finite number reaches no token that does not see it."""
    rng = np.random.default_rng(ntok + hd)
    q, cache, pos, counts, sees, cap = case(rng, bits, 2, ntok, nq, nkv, hd, start, False, ntok <= 64)
    clean, bound = attention_on_gpu(bits, q, cache, pos, np.full(2, ntok), sees, nq, nkv, hd, 0.2, cap)
    bad = ntok // 2
    see = R.visible(ntok, int(pos[0]), ntok, cap, None if sees is None else [int(x) for x in sees[0]])[:, pos[0] + bad]
    for which in (1, 3):
        for size in (2.0 ** 100, 2.0 ** 119, 2.0 ** 120.5, 3.3e38):
            c = [a.copy() for a in cache]
            f = np.float32(size)
            c[which][0, :, pos[0] + bad] = f if bits == 8 else f.view(np.uint32) >> 16
            got = attend(gpu_ctx, bits, q, c, pos, counts, sees, nq, nkv, hd, 0.2, cap)
            assert (np.abs(got - clean)[1] <= bound[1]).all()
            assert (np.abs(got - clean)[0, ~see] <= bound[0, ~see]).all(), (which, size)


@pytest.mark.parametrize("hd,nq,nkv,batch", [(64, 2, 2, 1), (128, 8, 2, 2), (64, 32, 32, 12), (128, 48, 24, 16)])
@pytest.mark.parametrize("room", [0, 3000])
def test_attention_of_one_position_rounds_its_v_to_nearest(gpu_ctx, hd, nq, nkv, batch, room):
    """Zero queries, one visible position, and a V head of a single code 1: what comes out is the V scale over 8, every
    step exact but for the scale's two pieces, 2^-23 of it, and their sum, a step at most."""
    rng = np.random.default_rng(hd + nq)
    ntok = 64
    cache = B.new_cache(8, batch, nkv, ntok + room, hd, rng)
    cache[2][:] = 0
    at = rng.integers(0, hd, cache[3].shape)
    np.put_along_axis(cache[2], at[..., None], 1, -1)
    cache[3][:] = rng.uniform(2.0 ** -6, 2.0 ** -3, cache[3].shape)
    sees = np.tile(np.uint64(1) << np.arange(ntok, dtype=np.uint64), (batch, 1))
    got = attend(gpu_ctx, 8, np.zeros((batch, ntok, nq, hd), np.float32), cache, np.zeros(batch, np.int32), None, sees, nq, nkv, hd, 0.17, ntok + room)
    vs = np.repeat(cache[3][:, :, :ntok].astype(np.float64), nq // nkv, 1).transpose(0, 2, 1)[..., None]  # [batch][ntok][nq][1]
    where = np.repeat(at[:, :, :ntok], nq // nkv, 1).transpose(0, 2, 1)[..., None] // 64 == np.arange(hd) // 64
    assert (got[~where] == 0).all()
    off = (np.abs(np.abs(got) * 8 - vs) / vs)[where]
    assert off.max() <= 2.0 ** -23 + 2.0 ** -23, off.max()


def test_keep_of_millions_of_heads_and_long_lists(gpu_ctx):
    """More than 2^21 (layer, row, head) triples, lists of 1024 entries: first positions that take the second one's codes and scales."""
    layers, rows, nkv, cap, n_keep = 3, 1000, 1024, 2, 1024
    g = torch.Generator(device="cuda").manual_seed(4)
    heads = layers * rows * nkv
    assert heads > 1 << 21
    c = [torch.randint(0, 256, (heads * cap, 32), generator=g, device="cuda", dtype=torch.uint8) for _ in range(2)]
    s = [torch.randint(0, 1 << 14, (heads * cap,), generator=g, device="cuda", dtype=torch.int16) for _ in range(2)]
    old = [t.clone() for t in (c[0], s[0], c[1], s[1])]
    keep = torch.full((rows, n_keep), -1, dtype=torch.int32, device="cuda")
    keep[:, 0] = 1
    keep[:, 1] = 1023  # (outside the cache)
    counts = torch.full((rows,), n_keep, dtype=torch.int32, device="cuda")
    counts[::7] = 0
    gpu_ctx.kv_keep(4, k2t.KVRows(c[0], s[0], c[1], s[1], cap=cap), torch.zeros(rows, dtype=torch.int32, device="cuda"), keep, n_keep, counts,
                    n_keep, layers, rows, nkv, 64)
    gpu_ctx.sync()
    moved = (counts > 0).view(1, rows, 1, 1)
    for got, was in zip((c[0], s[0], c[1], s[1]), old):
        got, was = (t.view(layers, rows, nkv, cap, -1) for t in (got, was))
        assert torch.equal(got[:, :, :, 1], was[:, :, :, 1])
        assert torch.equal(got[:, :, :, 0], torch.where(moved, was[:, :, :, 1], was[:, :, :, 0]))


@pytest.mark.parametrize("in_place", [False, True])
def test_logits_of_lists_without_entries(gpu_ctx, in_place):
    """Penalties of a history without tokens, beside no biases or some, and mask rows without masks."""
    rng = np.random.default_rng(9)
    rows, vocab = 3, 5001
    x = rng.standard_normal((rows, vocab + 3)).astype(np.float32)
    none = dict(history=np.zeros((rows, 0), np.int32), repeat=np.full(rows, 1.5, np.float32), presence=np.full(rows, 2.0, np.float32),
                history_len=np.full(rows, 4, np.int32), prompt_len=np.zeros(rows, np.int32),
                bias_tokens=np.zeros((rows, 0), np.int32), bias=np.zeros((rows, 0), np.float32),
                mask=np.zeros((0, 157), np.int32), mask_row=np.zeros(rows, np.int32))
    got = adjust(gpu_ctx, x, vocab, none, in_place)
    assert got[:, :vocab].tobytes() == x[:, :vocab].tobytes()
    some = dict(none, bias_tokens=np.array([[7, 5000], [1, 1], [-1, 6000]], np.int32), bias=rng.standard_normal((rows, 2)).astype(np.float32))
    want = R.logits(x, vocab, {k: some[k] for k in ("bias_tokens", "bias")})
    assert np.array_equal(adjust(gpu_ctx, x, vocab, some, in_place)[:, :vocab], want[:, :vocab])
