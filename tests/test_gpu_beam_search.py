"""GPU tests of the beam search on the device decoder: prompts, forked and
reordered caches, attention over shared pages and the selection run together,
against a search that keeps every continuation as a prompt of its own.

Logits of the two routes (a cache extended token by token, a prompt prefilled
anew) agree to 1e-4 per step, as the decoder's own tests hold them, so the
accumulated scores of n steps to n x 2e-4."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

SMALL = dict(num_layers=2, hidden=256, intermediate=512, vocab=1024, n_q_heads=4, n_kv_heads=2, head_dim=64,
             rms_eps=1e-6, rope_theta=1e6)


def make_model(sa, rows, max_pos, seed):
    m = sa.Qwen3(rows, max_pos, **SMALL)
    m.init_random(seed, 0.1)
    return m


def make_cache(sa, rows, tokens, dtype, spare=0):
    per = (tokens + 63) // 64
    return sa.KVCache(SMALL["num_layers"], SMALL["n_kv_heads"], SMALL["head_dim"], rows, per, rows * per + spare, dtype)


def last_logits(sa, model, paths):
    """Logits behind each path (all of one length), every path prefilled anew."""
    cache = make_cache(sa, len(paths), len(paths[0]), sa.SA_DTYPE_F32)
    for r, p in enumerate(paths):
        cache.reserve(r, len(p))
    out = torch.empty(len(paths), SMALL["vocab"], device="cuda")
    model.prefill(cache, torch.tensor(paths, dtype=torch.int32, device="cuda"), logits=out)
    torch.cuda.synchronize()
    cache.close()
    return torch.log_softmax(out.double(), -1).cpu()


def reference_search(sa, model, prompt, B, n_tokens, eos):
    beams, done = [(0.0, list(prompt))], []
    for n in range(1, n_tokens + 1):
        lp = last_logits(sa, model, [p for _, p in beams])
        cand = sorted(((s + float(lp[b, t]), b, t) for b, (s, _) in enumerate(beams)
                       for t in torch.topk(lp[b], 2 * B).indices.tolist()), key=lambda c: (-c[0], c[1], c[2]))[:2 * B]
        kept = []
        for rank, (s, b, t) in enumerate(cand):
            if eos is not None and t == eos:
                if rank < B:
                    done.append((s, beams[b][1] + [t]))
            elif len(kept) < B:
                kept.append((s, beams[b][1] + [t]))
        beams = kept
        ended = sorted((s for s, _ in done), reverse=True)[:B]
        if len(ended) == B and ended[-1] >= kept[0][0]:
            break
    return [(s, p[len(prompt):]) for s, p in sorted(done + beams, key=lambda x: -x[0])[:B]]


@pytest.mark.parametrize("G,B,L,n,eos", [(1, 4, 70, 9, None), (2, 3, 64, 8, None), (1, 1, 5, 6, None), (3, 2, 30, 40, 7),
                                         (1, 8, 130, 5, None)])
def test_search(sa, G, B, L, n, eos):
    model = make_model(sa, max(G * B, G), L + n + 1, 11 + B)
    cache = make_cache(sa, G * B, L + n, sa.SA_DTYPE_F32)
    gen = torch.Generator(device="cuda").manual_seed(L)
    prompts = torch.randint(0, SMALL["vocab"], (G, L), dtype=torch.int32, device="cuda", generator=gen)
    if eos is not None:      # a token that the search meets: the likeliest second one of the first prompt
        lp = last_logits(sa, model, [prompts[0].tolist()])
        eos = int(last_logits(sa, model, [prompts[0].tolist() + [int(lp[0].argmax())]])[0].argmax())
    got = model.beam_search(cache, prompts, B, n, eos)
    for g in range(G):
        want = reference_search(sa, model, prompts[g].tolist(), B, n, eos)
        assert [p for _, p in got[g]] == [p for _, p in want], (got[g], want)
        for (a, p), (b, _) in zip(got[g], want):
            assert abs(a - b) <= 2e-4 * len(p)
    cache.close()
    model.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("G,B,P", [(1, 4, 4100), (2, 8, 1000), (1, 20, 700), (2, 2, 300)])
def test_step_over_shared_pages(sa, dtype, G, B, P):
    """beam_step on forked rows (enough shared tokens for the shared attention,
    but for the last) against decode_step on rows with pages of their own."""
    dt = sa.SA_DTYPE_BF16 if dtype == "bf16" else sa.SA_DTYPE_F32
    rows, layers, Hkv, D, V = G * B, 2, 2, 64, SMALL["vocab"]
    model = make_model(sa, rows, P + 100, 3)
    plain, forked = (make_cache(sa, rows, P + 80, dt) for _ in range(2))
    gen = torch.Generator(device="cuda").manual_seed(P)
    for g in range(G):
        n = P - 7 * g
        kv = [[torch.randn(1, n, Hkv, D, device="cuda", generator=gen) for _ in range(2)] for _ in range(layers)]
        for cache, some in ((plain, range(g * B, g * B + B)), (forked, [g * B])):
            for r in some:
                cache.reserve(r, n)
                for layer in range(layers):
                    cache.append(layer, None, *kv[layer], seq_ids=[r])
                cache.commit(n, seqs=[r])
        for r in range(g * B + 1, g * B + B):
            forked.fork(r, g * B, n)
    scores = -5 * torch.rand(G, B, device="cuda", generator=gen)
    for step in range(3):
        tokens = torch.randint(0, V, (G, B), dtype=torch.int32, device="cuda", generator=gen)
        for r in range(rows):
            for cache in (plain, forked):
                cache.reserve(r, cache.length(r) + 1)
        logits = torch.empty(rows, V, device="cuda")
        model.decode_step(plain, tokens.view(-1), logits=logits)
        got = model.beam_step(forked, tokens, scores, 6)
        lp = torch.log_softmax(logits.double(), -1).view(G, B, V) + scores.double()[..., None]
        at = got[2].long() * V + got[1].long()
        assert (torch.gather(lp.view(G, -1), 1, at) - got[0].double()).abs().max() <= 2e-4
        # nothing better was left out
        best = torch.topk(lp.view(G, -1), 6).values
        assert (best - got[0].double()).abs().max() <= 2e-4
        parents = [g * B + (b + step) % B for g in range(G) for b in range(B)]
        for cache in (plain, forked):
            cache.reorder(range(rows), parents)
        assert [plain.length(r) for r in range(rows)] == [forked.length(r) for r in range(rows)]
    for r in range(rows):
        for layer in range(layers):
            a, b = (torch.stack(c.gather(layer, r, c.length(r))) for c in (plain, forked))
            assert torch.equal(a[..., :P // 64 * 64 - 64, :], b[..., :P // 64 * 64 - 64, :])
            assert (a - b).abs().max() <= (2e-4 if dtype == "f32" else 0.04)
    plain.close()
    forked.close()
    model.close()


def test_refusals(sa):
    model = make_model(sa, 4, 100, 5)
    cache = make_cache(sa, 4, 64, sa.SA_DTYPE_F32)
    lib = sa.lib()
    tok = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    sc = torch.zeros(1, 4, device="cuda")
    o = torch.full((1, 8), 7.0, device="cuda")
    i = torch.full((2, 8), 7, dtype=torch.int32, device="cuda")

    def call(m=model.handle, c=cache.handle, t=tok.data_ptr(), G=1, B=4, s=sc.data_ptr(), n=8, o=o.data_ptr()):
        return lib.sa_qwen3_beam_step(m, c, t, G, B, s, n, o, i.data_ptr(), i.data_ptr() + 32, None)

    for bad in (dict(m=None), dict(c=None), dict(t=None), dict(s=None), dict(o=None), dict(n=0), dict(n=65)):
        assert call(**bad) == sa.SA_EINVAL, bad
    for bad in (dict(G=0), dict(B=0), dict(B=5), dict(G=2), dict(G=1 << 20, B=1 << 20)):
        assert call(**bad) == sa.SA_ERANGE, bad
    assert call() == sa.SA_EFULL                      # nothing reserved
    for r in range(4):
        cache.reserve(r, 64)
    cache.set_len(0, 64)
    cache.fork(1, 0, 64)
    cache.set_len(1, 10)                              # back into the shared page
    cache.set_len(0, 10)
    assert call() == sa.SA_EINVAL and b"shares" in lib.sa_last_error()
    torch.cuda.synchronize()
    assert (o == 7).all() and [cache.length(r) for r in range(4)] == [10, 10, 0, 0]
    with pytest.raises(ValueError):
        model.beam_step(cache, tok.long(), sc, 8)
    with pytest.raises(ValueError):
        model.beam_step(cache, tok, sc[:, :2], 8)
    cache.close()
    model.close()


def test_one_probability_left(sa):
    """Beams of probability 0 stay unselected through the steps."""
    model = make_model(sa, 3, 100, 6)
    cache = make_cache(sa, 3, 64, sa.SA_DTYPE_F32)
    cache.reserve(0, 20)
    logits = torch.empty(1, SMALL["vocab"], device="cuda")
    model.prefill(cache, torch.arange(20, dtype=torch.int32, device="cuda")[None], logits=logits)
    cache.reorder(range(3), [0, 0, 0])
    for r in range(3):
        cache.reserve(r, 21)
    scores = torch.tensor([[-math.inf, -1.0, -math.inf]], device="cuda")
    s, t, b = model.beam_step(cache, torch.tensor([[1, 2, 3]], dtype=torch.int32, device="cuda"), scores, 5)
    assert (b == 1).all() and torch.isfinite(s).all() and (s.diff() <= 0).all()
    cache.close()
    model.close()


@pytest.mark.parametrize("P", [200, 4100])
def test_captured_steps_outlive_larger_ones(sa, P):
    """A beam step and a decode step captured into graphs, then steps of more
    rows, pages and selections, which need larger workspaces, and new tensors
    where a freed workspace would be: the graphs' replays still give what the
    eager steps gave, and leave the new tensors alone."""
    model = make_model(sa, 16, 9000, 8)
    small, large = make_cache(sa, 4, P + 80, sa.SA_DTYPE_F32), make_cache(sa, 16, 8800, sa.SA_DTYPE_F32)
    gen = torch.Generator(device="cuda").manual_seed(P)

    def fill(cache, rows, n):
        cache.reserve(0, n)
        for layer in range(SMALL["num_layers"]):
            kv = (torch.randn(1, n, 2, 64, device="cuda", generator=gen) for _ in range(2))
            cache.append(layer, None, *kv, seq_ids=[0])
        cache.commit(n, seqs=[0])
        for r in range(1, rows):
            cache.fork(r, 0, n)
        for r in range(rows):
            cache.reserve(r, n + 1)

    fill(small, 4, P)
    tokens = torch.tensor([[5, 6, 7, 8]], dtype=torch.int32, device="cuda")
    scores = torch.tensor([[-1.0, -2.0, -1.5, -0.5]], device="cuda")
    out = (torch.empty(1, 6, device="cuda"), *(torch.empty(1, 6, dtype=torch.int32, device="cuda") for _ in range(2)))
    logits = torch.empty(4, SMALL["vocab"], device="cuda")

    def back(cache, rows, n):
        for r in range(rows):
            cache.set_len(r, n)
        torch.cuda.synchronize()

    steps = (lambda: model.beam_step(small, tokens, scores, 6, out=out),
             lambda: model.decode_step(small, tokens.view(-1), logits=logits))
    want, graphs = [], []
    for step in steps:
        step()
        torch.cuda.synchronize()
        want.append([t.clone() for t in (*out, logits)])
        back(small, 4, P)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            step()
        back(small, 4, P)
    fill(large, 16, 8700)
    model.beam_step(large, torch.arange(16, dtype=torch.int32, device="cuda").view(2, 8), torch.zeros(2, 8, device="cuda"), 64)
    back(large, 16, 8700)
    model.decode_step(large, torch.arange(16, dtype=torch.int32, device="cuda"))
    fresh = [torch.full((1 << n,), 0xa5, dtype=torch.uint8, device="cuda") for n in range(12, 27) for _ in range(2)]
    for rep in range(3):
        for graph, w, some in zip(graphs, want, (slice(0, 3), slice(3, 4))):
            for t in (*out, logits):
                t.fill_(9)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip((*out, logits)[some], w[some])), rep
            back(small, 4, P)
    assert all((t == 0xa5).all() for t in fresh)
    del graphs
    for c in (small, large):
        c.close()
    model.close()


@pytest.mark.parametrize("Hq,Hkv", [(6, 2), (16, 1), (5, 1)])
@pytest.mark.parametrize("P", [70, 4100])
def test_head_ratios(sa, Hq, Hkv, P):
    """Head ratios that the row-by-row attention has no kernel for, behind short
    and long prompts, against the paths prefilled anew."""
    desc = dict(SMALL, n_q_heads=Hq, n_kv_heads=Hkv)
    model = sa.Qwen3(4, P + 10, **desc)
    model.init_random(9, 0.1)
    per = P // 64 + 1

    def cache_of(rows):
        return sa.KVCache(desc["num_layers"], Hkv, 64, rows, per, rows * per, sa.SA_DTYPE_F32)

    gen = torch.Generator(device="cuda").manual_seed(P)
    prompt = torch.randint(0, SMALL["vocab"], (1, P), dtype=torch.int32, device="cuda", generator=gen)
    cache = cache_of(4)
    cache.reserve(0, P)
    model.prefill(cache, prompt)
    cache.reorder(range(4), [0] * 4)
    for r in range(4):
        cache.reserve(r, P + 2)
    tokens = torch.tensor([[3, 900, 17, 4]], dtype=torch.int32, device="cuda")
    scores = torch.tensor([[-1.0, -3.0, -2.0, -1.5]], device="cuda")
    got = model.beam_step(cache, tokens, scores, 6)
    paths = torch.cat([prompt.expand(4, P), tokens.view(4, 1)], 1)
    anew = cache_of(4)
    for r in range(4):
        anew.reserve(r, P + 1)
    logits = torch.empty(4, SMALL["vocab"], device="cuda")
    model.prefill(anew, paths.contiguous(), logits=logits)
    lp = torch.log_softmax(logits.double(), -1).view(1, 4, -1) + scores.double()[..., None]
    at = got[2].long() * SMALL["vocab"] + got[1].long()
    assert (torch.gather(lp.view(1, -1), 1, at) - got[0].double()).abs().max() <= 2e-4
    assert (torch.topk(lp.view(1, -1), 6).values - got[0].double()).abs().max() <= 2e-4
    # the ordinary step has no kernel for them and says so before it does anything
    with pytest.raises(RuntimeError, match="n_q_heads"):
        model.decode_step(cache, tokens.view(-1))
    assert [cache.length(r) for r in range(4)] == [P + 1] * 4
    for c in (cache, anew):
        c.close()
    model.close()


def test_step_in_place(sa):
    """A step whose results take the scores' place."""
    model = make_model(sa, 6, 100, 10)
    gen = torch.Generator(device="cuda").manual_seed(1)
    tokens = torch.randint(0, SMALL["vocab"], (2, 3), dtype=torch.int32, device="cuda", generator=gen)
    got = []
    for apart in (True, False):
        cache = make_cache(sa, 6, 64, sa.SA_DTYPE_F32)
        for r in range(6):
            cache.reserve(r, 21)
        model.prefill(cache, torch.arange(120, dtype=torch.int32, device="cuda").view(6, 20))
        scores = torch.tensor([[-1.0, -2.0, -0.5], [-3.0, -0.1, -2.5]], device="cuda")
        out = (torch.empty(2, 3, device="cuda") if apart else scores,
               *(torch.empty(2, 3, dtype=torch.int32, device="cuda") for _ in range(2)))
        model.beam_step(cache, tokens, scores, 3, out=out)
        got.append(out)
        torch.cuda.synchronize()
        if not apart:
            with pytest.raises(RuntimeError, match="out_scores"):
                wide = torch.zeros(12, device="cuda")
                model.beam_step(cache, tokens, wide[:6].view(2, 3), 6,
                                out=(wide.view(2, 6), *(torch.empty(2, 6, dtype=torch.int32, device="cuda") for _ in range(2))))
            assert [cache.length(r) for r in range(6)] == [21] * 6
        cache.close()
    assert all(torch.equal(a, b) for a, b in zip(*got))
    model.close()
