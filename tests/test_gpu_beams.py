"""k2t_model_beam_search against the model's own one-sequence steps, and the operators it is made of run
together as a program would.

Bar: two paths of one model may differ by 2e-2 of the largest logit (the end-to-end bar of the decode
tests: a last-ulp difference can move an int8 code), so a log probability by twice that, and a score of
n tokens by n times as much."""
import numpy as np
import pytest
import torch

import branch_ref as R
import k2t
from k2tb_writer import random_moe_layer, write_k2tm
from model_oracle import quantize_matrix, random_model
from test_gpu_model import P55454, TINY, TINY128, _close, _gpu_model

pytestmark = pytest.mark.gpu


def log_probs(logits):
    x = logits.astype(np.float64)
    x = x - x.max()
    return x - np.log(np.exp(x).sum())


def follow(gm, prompt, first, tokens):
    """Logits of every step of a given continuation, one sequence at a time."""
    gm.reset()
    gm.prefill(np.array(prompt, np.int32), want_logits=False)
    out = [gm.decode(int(first))]
    for t in tokens[:-1]:
        out.append(gm.decode(int(t)))
    return out


def search(gm, prompt, first, n_beams, n_steps, eos=-1):
    gm.reset()
    gm.prefill(np.array(prompt, np.int32), want_logits=False)
    return gm.beam_search(first, n_beams, n_steps, eos)


def check_search(gm, prompt, first, n_beams, n_steps, eos=-1):
    tokens, scores = search(gm, prompt, first, n_beams, n_steps, eos)
    pos = gm.position()
    assert (np.diff(scores) <= 0).all()
    assert len({tuple(t) for t in tokens}) == n_beams
    after = gm.decode(int(tokens[0][-1])) if eos < 0 else None
    for t, s in zip(tokens, scores):
        steps = follow(gm, prompt, first, t)
        bar = 4e-2 * max(np.abs(x).max() for x in steps)
        n = n_steps
        if eos >= 0 and eos in t:
            n = int(np.argmax(t == eos)) + 1
            assert (t[n:] == eos).all()
        want = sum(log_probs(x)[k] for x, k in list(zip(steps, t))[:n])
        assert abs(s - want) <= n * bar + 1e-4, (s, want, bar)
    # the cache and the position afterwards are those of the best beam
    fed = n_steps - 1 if eos < 0 or eos not in tokens[0][:-1] else int(np.argmax(tokens[0] == eos))
    assert pos == len(prompt) + 1 + fed
    if after is not None:
        steps = follow(gm, prompt, first, list(tokens[0]) + [0])
        ok, info = _close(after, steps[-1], 0.9999)
        assert ok, info
    return tokens, scores


@pytest.mark.parametrize("name,cfg,fmt,planes,bits", [("nf4", TINY, "nf4", None, 8), ("p55454", TINY, "n4", P55454, 4),
                                                      ("b6_hd128", TINY128, "n4", {k: 6 for k in P55454}, 8),
                                                      ("nf4_hd128", TINY128, "nf4", None, 4)])
@pytest.mark.parametrize("n_beams", [1, 4, 19])
def test_search_scores_and_state(gpu_ctx, name, cfg, fmt, planes, bits, n_beams):
    print(f"beam search {name} kv {bits} beams {n_beams}", flush=True)
    layers, head, fn = random_model(cfg, seed=5, fmt=fmt, planes=planes)
    gm, _ = _gpu_model(gpu_ctx, cfg, layers, head, fn, max_batch=20)
    gm.set_kv_bits(bits)
    check_search(gm, [3, 9, 250, 17, 4], 77, n_beams, 6)


def test_search_finds_the_best(gpu_ctx):
    """As many beams as candidates that could matter: two steps of the 64 best first tokens hold the
    best pairs, which are found by going through every first token."""
    cfg = dict(TINY, vocab=72)
    layers, head, fn = random_model(cfg, seed=8, fmt="nf4")
    gm, _ = _gpu_model(gpu_ctx, cfg, layers, head, fn, max_batch=64)
    prompt, first = [5, 60, 33], 12
    tokens, scores = search(gm, prompt, first, 64, 2)
    step0 = follow(gm, prompt, first, [0])[0]
    lp0, bar = log_probs(step0), 0.0
    pairs = []
    for a in range(72):
        logits = follow(gm, prompt, first, [a, 0])[1]
        bar = max(bar, 4e-2 * max(np.abs(logits).max(), np.abs(step0).max()))
        pairs += [(lp0[a] + p, a, b) for b, p in enumerate(log_probs(logits))]
    pairs.sort(reverse=True)
    want = np.array([p[0] for p in pairs[:64]])
    assert np.abs(scores - want).max() <= 2 * bar + 1e-4
    assert tuple(tokens[0]) in {p[1:] for p in pairs if p[0] >= pairs[0][0] - 2 * bar}


def test_one_beam_is_greedy_and_repeats(gpu_ctx):
    layers, head, fn = random_model(TINY, seed=2, fmt="nf4")
    gm, _ = _gpu_model(gpu_ctx, TINY, layers, head, fn, max_batch=4)
    prompt, first = [1, 2, 3], 44
    tokens, scores = search(gm, prompt, first, 1, 8)
    for x, t in zip(follow(gm, prompt, first, tokens[0]), tokens[0]):
        assert x[t] >= x.max() - 4e-2 * np.abs(x).max()
    again = search(gm, prompt, first, 1, 8)
    assert np.array_equal(again[0], tokens) and np.array_equal(again[1], scores)
    # other sizes in between, and a second search behind the first: the same sizes again, the same result
    search(gm, prompt, first, 4, 11)
    gm.beam_search(7, 3, 5)
    again = search(gm, prompt, first, 1, 8)
    assert np.array_equal(again[0], tokens) and np.array_equal(again[1], scores)


def test_eos_ends_beams(gpu_ctx):
    layers, head, fn = random_model(TINY, seed=6, fmt="nf4")
    gm, _ = _gpu_model(gpu_ctx, TINY, layers, head, fn, max_batch=8)
    prompt, first = [8, 100], 31
    free, _ = check_search(gm, prompt, first, 5, 7)
    for eos in (int(free[0][0]), int(free[0][2]), int(free[1][-1])):
        tokens, _ = check_search(gm, prompt, first, 5, 7, eos)
        assert any(eos in t for t in tokens)


def test_a_search_whose_beams_all_end(gpu_ctx):
    """Two beams over two tokens of one embedding, so that the same one is the more probable behind the
    prompt and behind the other: as eos it ends both beams in two steps, and a longer search is that and eos."""
    cfg = dict(TINY, vocab=2, max_seq=80)
    layers, head, fn = random_model(cfg, seed=10, fmt="nf4")
    gm, _ = _gpu_model(gpu_ctx, cfg, layers, head, fn, max_batch=2)
    gm.set_embedding(k2t.EMBED_F32, rows=np.tile(np.random.default_rng(3).standard_normal(256).astype(np.float32), (2, 1)))
    tried = 0
    for prompt in ([0], [1], [0, 1], [1, 1], [0, 0, 1], [1, 0, 1], [1, 1, 0], [0, 0, 0]):
        a = follow(gm, prompt, 1, [0])[0]
        eos = int(a.argmax())
        b = follow(gm, prompt, 1, [1 - eos, 0])[1]
        if min(a[eos] - a[1 - eos], b[eos] - b[1 - eos]) < 8e-2 * max(np.abs(a).max(), np.abs(b).max()):
            continue  # (not told apart by two paths of the model, or the other token)
        tried += 1
        tokens, scores = check_search(gm, prompt, 1, 2, 60, eos)
        want = np.full((2, 60), eos)
        want[1, 0] = 1 - eos
        assert np.array_equal(tokens, want)
        for n_steps in (2, 3, 17, 18, 19, 60):
            t, s = search(gm, prompt, 1, 2, n_steps, eos)
            assert np.array_equal(t, want[:, :n_steps]) and np.array_equal(s, scores)
            assert gm.position() == len(prompt) + 1
    assert tried


def test_more_beams_than_tokens(gpu_ctx):
    """The first step has fewer candidates than beams: rows that are not in use, and used ones later."""
    cfg = dict(TINY, vocab=24)
    layers, head, fn = random_model(cfg, seed=9, fmt="nf4")
    gm, _ = _gpu_model(gpu_ctx, cfg, layers, head, fn, max_batch=33)
    tokens, scores = search(gm, [1, 2], 3, 33, 1)
    assert sorted(tokens[:24, 0]) == list(range(24)) and (scores[24:] == -np.inf).all() and np.isfinite(scores[:24]).all()
    check_search(gm, [1, 2], 3, 33, 3)


def test_long_prompt_and_limits(gpu_ctx):
    """A prompt past the single-launch attention, up to the last position the cache holds."""
    cfg = dict(TINY128, n_layers=1, max_seq=900)
    layers, head, fn = random_model(cfg, seed=4, fmt="nf4")
    gm, _ = _gpu_model(gpu_ctx, cfg, layers, head, fn, max_batch=64)
    prompt = np.random.default_rng(0).integers(0, cfg["vocab"], 890)
    check_search(gm, prompt, 5, 3, 9)  # (one more position than check_search's own step needs)
    gm.reset()
    gm.prefill(prompt.astype(np.int32), want_logits=False)
    tokens, _ = gm.beam_search(5, 3, 10)
    assert gm.position() == 900 and tokens.shape == (3, 10)
    for bad in (dict(n_beams=0), dict(n_beams=65), dict(n_steps=0), dict(eos=cfg["vocab"]), dict(eos=-2), dict(first_token=-1),
                dict(n_steps=2)):  # (the last: past max_seq)
        a = dict(first_token=1, n_beams=2, n_steps=1, eos=-1)
        a.update(bad)
        with pytest.raises(k2t.K2TError) as e:
            gm.beam_search(**a)
        assert e.value.code == -1
    few = np.zeros(64, np.int32)  # (refused before anything is written)
    assert k2t.lib().k2t_model_beam_search(gm.h, 1, 2, 2 ** 31 - 1, -1, few.ctypes.data, few.ctypes.data) == -1
    gm.reset()
    gm.set_exact(True)
    with pytest.raises(k2t.K2TError, match="fast mode"):
        gm.beam_search(1, 2, 2)
    gm.set_exact(False)
    gm.set_kv_window(64, 4)
    with pytest.raises(k2t.K2TError, match="full KV cache"):
        gm.beam_search(1, 2, 2)


def test_mixture_of_experts_model(gpu_ctx):
    """Sparse-MoE layers, QK-norm, q_dim != hidden: rows of a step grouped by expert."""
    cfg = dict(n_layers=2, hidden=256, n_heads=4, n_kv_heads=2, head_dim=128, intermediate=64, vocab=300, max_seq=40,
               rms_eps=1e-6, rope_theta=10000.0)
    rng = np.random.default_rng(5)
    d, E, k, dff, hd = 256, 16, 4, 128, 128
    moe = [random_moe_layer(rng, d, dff, E, bits=3) for _ in range(2)]
    bank = k2t.ExpertBank.upload(gpu_ctx, write_k2tm([m[0] for m in moe], d, dff, 3, 2))
    gm = k2t.Model(gpu_ctx, cfg, max_batch=8)
    up = lambda r, c: (lambda m: gpu_ctx.upload_nf(m.rows, m.cols, 4, m.sgc, m.cb, m.pair, m.tail))(  # noqa: E731
        quantize_matrix((rng.standard_normal((r, c)) * 0.02).astype(np.float32), "nf4"))
    norm = lambda n: (1 + 0.1 * rng.standard_normal(n)).astype(np.float32)  # noqa: E731
    mats = []
    for li in range(2):
        mats += [up(8 * hd, d), up(d, 4 * hd)]
        gm.set_layer(li, mats[-2], mats[-1], None, None, norm(d), norm(d))
        gm.set_qk_norm(li, norm(hd), norm(hd))
        gm.set_moe(li, bank, li, moe[li][1], k, True, 0)
    mats.append(up(300, d))
    gm.set_head(mats[-1], norm(d))
    for n_beams in (1, 6):
        check_search(gm, [3, 250, 17], 9, n_beams, 4)


@pytest.mark.parametrize("fmt,planes", [("nf4", None), ("n4", P55454)])
def test_search_beside_batched_gemvs_of_the_context(gpu_ctx, fmt, planes):
    """From 16 beams on a search's batched GEMVs read their activations in tiles. The context's scratch, into
    which a GEMV would copy them, belongs to calls on the context's stream: products queued there come out as
    they do alone, and so does a search that runs beside them."""
    cfg = dict(n_layers=1, hidden=1024, n_heads=16, n_kv_heads=4, head_dim=64, intermediate=1536, vocab=4096, max_seq=40,
               rms_eps=1e-5, rope_theta=10000.0)
    layers, head, fn = random_model(cfg, seed=3, fmt=fmt, planes=planes)
    gm, mats = _gpu_model(gpu_ctx, cfg, layers, head, fn, max_batch=48)
    mat, ntok = mats[-1], 512  # (the lm_head once more, for more tokens than the search has)
    gpu_ctx.set_stream(torch.cuda.Stream())
    try:
        g = torch.Generator(device="cuda").manual_seed(7)
        xq = torch.randint(-127, 128, (ntok, 1024), generator=g, device="cuda").to(torch.int8)
        xs = torch.rand(ntok, 16, generator=g, device="cuda") / 127
        xsum = xq.view(ntok, 16, 64).sum(-1, dtype=torch.int32)
        outs = [torch.empty(ntok, 4096, device="cuda") for _ in range(60)]
        torch.cuda.synchronize()
        gpu_ctx.gemv(mat, xq, xs, xsum, outs[0], ntok=ntok, out_stride=4096)
        gpu_ctx.sync()
        want = outs[0].clone()
        for n_beams in (16, 48):
            alone = search(gm, [3, 9, 250], 77, n_beams, 5)
            gpu_ctx.set_mfma(2)  # (the GEMVs' own copies)
            copied = search(gm, [3, 9, 250], 77, n_beams, 5)
            gpu_ctx.set_mfma(1)
            assert np.array_equal(copied[0], alone[0]) and np.array_equal(copied[1], alone[1])
            for o in outs:
                o.zero_()
            torch.cuda.synchronize()
            for o in outs:
                gpu_ctx.gemv(mat, xq, xs, xsum, o, ntok=ntok, out_stride=4096)
            beside = search(gm, [3, 9, 250], 77, n_beams, 5)
            gpu_ctx.sync()
            assert np.array_equal(beside[0], alone[0]) and np.array_equal(beside[1], alone[1])
            assert all(torch.equal(o, want) for o in outs)
    finally:
        gpu_ctx.sync()
        gpu_ctx.set_mfma(1)
        gpu_ctx.set_stream(torch.cuda.current_stream())


# ---------------------------------------------------------------- the operators in a row
class Program:
    """A step of beam search over one layer's worth of heads: append the rows' K / V, attend, choose,
    rearrange; everything on the device, positions and lengths included."""

    def __init__(self, ctx, bits, n_seq, beams, nq, nkv, hd, prefix, steps, vocab, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.ctx, self.bits, self.dims, self.steps, self.vocab = ctx, bits, (n_seq, beams, nq, nkv, hd), steps, vocab
        rows = n_seq * beams
        self.qkv = rnd(steps, rows, (nq + 2 * nkv) * hd)
        self.logits = 3 * rnd(steps, rows, vocab)
        self.in_qkv, self.in_logits = torch.empty_like(self.qkv[0]), torch.empty_like(self.logits[0])
        caches = []
        for r, cap in ((n_seq, prefix + 2), (rows, steps + 1)):
            codes = (r, nkv, cap, hd if bits == 8 else hd // 2)
            sc = (r, nkv, cap) if bits == 8 else (r, nkv, cap, hd // 64)
            kinds = ((codes, torch.int8 if bits == 8 else torch.uint8), (sc, torch.float32 if bits == 8 else torch.int16))
            caches.append([torch.zeros(s, dtype=d, device="cuda") for _ in "kv" for s, d in kinds])
        self.pre_t, self.tail_t = caches
        self.pos = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.len = torch.ones(rows, dtype=torch.int32, device="cuda")
        self.pre = k2t.KVRows(*self.pre_t, cap=prefix + 2, len=prefix)
        self.tail = k2t.KVRows(*self.tail_t, cap=steps + 1, len=steps, d_len=self.len)
        x = rnd(n_seq * prefix, 2 * nkv * hd)
        ctx.kv_append(bits, x, x.data_ptr() + 4 * nkv * hd, 2 * nkv * hd, n_seq, prefix, nkv, hd,
                      torch.zeros(n_seq, dtype=torch.int32, device="cuda"), self.pre)
        self.x = x
        self.scores = torch.zeros(rows, device="cuda")
        self.done, self.tok, self.par = (torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(3))
        self.out = torch.zeros(rows, nq * hd, device="cuda")
        self.ws_a = torch.zeros(ctx.attn_shared_workspace(n_seq, beams, nq, nkv, hd, prefix, steps), dtype=torch.uint8,
                                device="cuda")
        self.ws_s = torch.zeros(ctx.beam_select_workspace(n_seq, beams, vocab, beams), dtype=torch.uint8, device="cuda")

    def reset(self):
        self.pos.zero_()
        self.len.fill_(1)
        self.scores.zero_()
        self.scores.view(self.dims[0], -1)[:, 1:] = -float("inf")  # the first step starts from one row
        self.done.zero_()
        for t in self.tail_t:
            t.zero_()

    def step(self):
        n_seq, beams, nq, nkv, hd = self.dims
        c, width = self.ctx, (nq + 2 * nkv) * hd
        k = self.in_qkv.data_ptr() + 4 * nq * hd
        c.kv_append(self.bits, k, k + 4 * nkv * hd, width, n_seq * beams, 1, nkv, hd, self.pos, self.tail)
        c.attn_shared(self.bits, self.in_qkv, width, n_seq, beams, nq, nkv, hd, self.pre, self.tail, hd ** -0.5, self.out,
                      self.ws_a)
        c.beam_select(self.in_logits, self.vocab, self.vocab, self.scores, self.done, n_seq, beams, beams, 3, self.scores,
                      self.tok, self.par, self.done, self.ws_s)
        c.kv_reorder(self.bits, self.tail, self.par, 1, n_seq, beams, nkv, hd)
        self.pos += 1
        self.len += 1

    def run(self, step):
        """Every step with its inputs; what it leaves."""
        self.reset()
        seen = []
        for i in range(self.steps):
            self.in_qkv.copy_(self.qkv[i])
            self.in_logits.copy_(self.logits[i])
            step()
            seen.append([t.clone() for t in (self.out, self.scores, self.tok, self.par, self.done, *self.tail_t)])
        torch.cuda.synchronize()
        return seen


def same(a, b):
    return all(torch.equal(x, y) for s, t in zip(a, b) for x, y in zip(s, t))


@pytest.mark.parametrize("bits,hd", [(8, 64), (4, 128)])
def test_operators_in_a_row(gpu_ctx, bits, hd):
    """Five steps of two sequences of four beams against the references, on the same choices."""
    gpu_ctx.set_stream(torch.cuda.current_stream())
    n_seq, beams, nq, nkv, prefix, steps, vocab = 2, 4, 4, 2, 37, 5, 400
    p = Program(gpu_ctx, bits, n_seq, beams, nq, nkv, hd, prefix, steps, vocab, 1)
    seen = p.run(p.step)
    rows = n_seq * beams
    host = lambda t: t.cpu().numpy().view(np.uint16) if t.dtype == torch.int16 else t.cpu().numpy()  # noqa: E731
    pre = [host(t) for t in p.pre_t]
    tail = R.new_cache(bits, rows, nkv, steps + 1, hd)
    for a in tail:
        a[:] = 0
    scores = np.full(rows, -np.inf, np.float32)
    scores[::beams] = 0
    done = np.zeros(rows, np.int32)
    for i in range(steps):
        out, sc, tok, par, dn, *t = (host(x) for x in seen[i])
        qkv = host(p.qkv[i])
        for r in range(rows):
            for h in range(nkv):
                for w in range(2):
                    o = (nq + w * nkv + h) * hd
                    tail[2 * w][r, h, i], tail[2 * w + 1][r, h, i] = R.store(bits, qkv[r, o:o + hd])
        want, bound = R.attention(bits, qkv[:, :nq * hd].reshape(rows, nq, hd), pre, tail, [prefix] * n_seq, [i + 1] * rows,
                                  beams, nq, nkv, hd, hd ** -0.5)
        assert (np.abs(out.reshape(rows, nq, hd) - want) <= bound).all()
        ws, wt, wp, wd, gap = R.select(host(p.logits[i]), scores, done, n_seq, beams, beams, 3)
        assert gap > 2.0 ** -15
        assert np.array_equal(tok, wt.reshape(-1)) and np.array_equal(par, wp.reshape(-1)) and np.array_equal(dn, wd.reshape(-1))
        assert np.abs(sc - ws.reshape(-1)).max() <= 2.0 ** -18 + 2.0 ** -24 * np.abs(ws).max()
        scores, done = sc, dn
        tail = [np.concatenate([a[wp.reshape(-1), :, :i + 1], a[:, :, i + 1:]], 2) for a in tail]
        for g, a in zip(t, tail):
            assert np.array_equal(g, a)


def test_captured_steps_and_two_graphs_of_one_context(gpu_ctx):
    """A step captured once and replayed, with the program's own eager work and synchronizations between:
    every replay equals the eager step.  Two programs of one context, replayed in turn and overlapping on
    two streams: their workspaces are their own."""
    main = torch.cuda.current_stream()
    gpu_ctx.set_stream(main)
    ps = [Program(gpu_ctx, 8, 2, 4, 8, 2, 64, 900, 6, 5000, 3), Program(gpu_ctx, 4, 1, 8, 8, 2, 128, 700, 6, 9000, 4)]
    eager = [p.run(p.step) for p in ps]
    graphs = []
    for p in ps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            gpu_ctx.set_stream(torch.cuda.current_stream())
            p.step()
        gpu_ctx.set_stream(main)
        graphs.append(g)
    for p, g, e in zip(ps, graphs, eager):
        assert same(p.run(g.replay), e)
    assert same(ps[0].run(ps[0].step), eager[0])  # eager again, then the graphs once more
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    seen = [[], []]
    for p in ps:
        p.reset()
    torch.cuda.synchronize()
    for i in range(6):
        for j, (p, g) in enumerate(zip(ps, graphs)):
            with torch.cuda.stream(streams[j]):
                p.in_qkv.copy_(p.qkv[i])
                p.in_logits.copy_(p.logits[i])
                g.replay()
                seen[j].append([t.clone() for t in (p.out, p.scores, p.tok, p.par, p.done, *p.tail_t)])
    torch.cuda.synchronize()
    assert same(seen[0], eager[0]) and same(seen[1], eager[1])


def test_on_another_stream_than_the_contexts_first(gpu_ctx):
    """The calls run on the context's stream: work queued there before them is seen, a busy default
    stream is not waited for."""
    ctx = k2t.Ctx(0)
    s = torch.cuda.Stream()
    ctx.set_stream(s)
    with torch.cuda.stream(s):
        p = Program(ctx, 8, 1, 3, 6, 2, 64, 50, 3, 700, 9)
        a = p.run(p.step)
        b = p.run(p.step)
    torch.cuda.synchronize()
    assert same(a, b)
    gpu_ctx.set_stream(torch.cuda.current_stream())
    q = Program(gpu_ctx, 8, 1, 3, 6, 2, 64, 50, 3, 700, 9)
    assert same(q.run(q.step), a)
    ctx.close()
