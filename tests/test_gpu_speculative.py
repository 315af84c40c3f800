"""GPU tests of the decoder over chunks of new tokens (extend) and of generation
with drafted tokens, against the decoder's own single steps and prompts.

fp32 cache: the two compute the same sums in other orders: logits max-abs 1e-4 and
relative L2 1e-5, the bounds of the decoder's other tests, and equal greedy
tokens.  bf16 and 8-bit caches: a stored value may fall on the other side of a
rounding, the relative L2 bound is the one of the decoder's bf16 tests, 2e-2 (8 bits: a
step is 16 times as large, 2^-3 of a value against 2^-7, on the few values that
flip).
"""
from __future__ import annotations

import pytest
import torch

from kv_rows import code

pytestmark = pytest.mark.gpu

CFG = dict(num_layers=2, hidden=128, intermediate=192, vocab=256, n_q_heads=4, n_kv_heads=2, head_dim=64,
           rms_eps=1e-6, rope_theta=1e6)
CFG128 = dict(CFG, hidden=256, head_dim=128)


def make_model(sa, max_batch, max_pos, cfg=CFG, seed=5, std=0.1):
    model = sa.Qwen3(max_batch, max_pos, **cfg)
    model.init_random(seed, std)
    return model


def make_cache(sa, kv, rows, tokens, cfg=CFG):
    per = (tokens + 63) // 64
    cache = sa.KVCache(cfg["num_layers"], cfg["n_kv_heads"], cfg["head_dim"], rows, per, rows * per, code(sa, kv))
    for r in range(rows):
        cache.reserve(r, tokens)
    return cache


def tokens_of(n, seed, vocab=256):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, vocab, (n,), generator=g).int().cuda()


def by_steps(sa, model, kv, seqs, cfg=CFG):
    """Logits of every token of every sequence, each alone and token by token."""
    out = []
    for x in seqs:
        cache = make_cache(sa, kv, 1, len(x), cfg)
        rows = torch.empty(len(x), cfg["vocab"], device="cuda")
        for t in range(len(x)):
            model.decode_step(cache, x[t:t + 1].contiguous(), logits=rows[t:t + 1])
        out.append(rows)
    return out


def close(got, want, kv):
    rel = ((got - want).norm() / want.norm()).item()
    if kv == "f32":
        assert (got - want).abs().max().item() <= 1e-4 and rel <= 1e-5
        assert torch.equal(got.argmax(-1), want.argmax(-1))
    else:
        assert rel <= 2e-2, rel


@pytest.mark.parametrize("kv", ["f32", "bf16", "fp8"])
@pytest.mark.parametrize("cfg", [CFG, CFG128])
@pytest.mark.parametrize("max_batch", [8, 64, 512])
def test_chunks_equal_steps(sa, kv, cfg, max_batch):
    """Rounds of ragged chunks: few rows, up to max_batch (all logits), beyond it (the last ones')."""
    model = make_model(sa, max_batch, 300, cfg)
    rounds = [[3, 1, 2], [1, 4, 2], [2, 1, 1], [40, 65, 130], [1, 1, 1]]
    seqs = [tokens_of(sum(r[i] for r in rounds), i) for i in range(3)]
    want = by_steps(sa, model, kv, seqs, cfg)
    cache = make_cache(sa, kv, 3, 300, cfg)
    at = [0, 0, 0]
    for counts in rounds:
        x = torch.cat([s[a:a + n] for s, a, n in zip(seqs, at, counts)]).contiguous()
        every = sum(counts) <= max_batch
        logits = torch.empty(sum(counts) if every else 3, cfg["vocab"], device="cuda")
        new = model.extend(cache, x, counts, all_rows=every, logits=logits)
        rows = [w[a:a + n] if every else w[a + n - 1:a + n] for w, a, n in zip(want, at, counts)]
        close(logits, torch.cat(rows), kv)
        assert torch.equal(new.long(), logits.argmax(-1))
        last = torch.empty(3, cfg["vocab"], device="cuda")
        for i in range(3):
            at[i] += counts[i]
        assert [cache.length(i) for i in range(3)] == at
        if every:       # the same without the others' logits
            cache.set_lens(range(3), [a - n for a, n in zip(at, counts)])
            only = model.extend(cache, x, counts, logits=last)
            ends = torch.tensor(counts).cumsum(0) - 1
            close(last, logits[ends.cuda()], "f32")
            assert torch.equal(only, new[ends.cuda()])


@pytest.mark.parametrize("kv", ["f32", "fp8"])
def test_a_prompt_in_chunks_equals_a_prompt(sa, kv):
    model = make_model(sa, 2, 400, CFG128)
    x = tokens_of(2 * 390, 3).view(2, 390)
    a, b = (make_cache(sa, kv, 2, 400, CFG128) for _ in range(2))
    want = torch.empty(2, 256, device="cuda")
    model.prefill(a, x, logits=want)
    got = torch.empty_like(want)
    for lo, hi in ((0, 150), (150, 389), (389, 390)):
        model.extend(b, x[:, lo:hi].contiguous(), logits=got)
    # a prompt attends over its keys and values as they are, a chunk as they are held:
    # in 8 bits they differ by up to 2^-4 each
    rel = ((got - want).norm() / want.norm()).item()
    assert rel <= (1e-5 if kv == "f32" else 2.0 ** -3)
    if kv == "f32":
        assert (got - want).abs().max().item() <= 1e-4
    for r in range(2):
        for p, q in zip(a.gather(0, r, 390), b.gather(0, r, 390)):   # layer 0 has one input
            assert (p - q).norm().item() <= 1e-2 * p.norm().item()


def test_rejected_tokens_leave_no_trace(sa):
    """Tokens appended without a commit are overwritten by what comes instead."""
    model = make_model(sa, 16, 200)
    x = tokens_of(120, 4)
    cache = make_cache(sa, "f32", 1, 200)
    model.extend(cache, x[:60].contiguous(), [60])
    model.extend(cache, tokens_of(10, 9), [10], all_rows=True, commit=False)
    assert cache.length(0) == 60
    model.extend(cache, x[60:63].contiguous(), [3], all_rows=True, commit=False)
    cache.set_lens([0], [62])
    logits = torch.empty(1, 256, device="cuda")
    model.extend(cache, x[62:120].contiguous(), [58], logits=logits)
    close(logits, by_steps(sa, model, "f32", [x])[0][-1:], "f32")


def test_sequences_without_new_tokens(sa):
    model = make_model(sa, 16, 100)
    cache = make_cache(sa, "f32", 3, 100)
    x = tokens_of(8, 6)
    model.extend(cache, x[:3].contiguous(), [0, 3, 0], all_rows=True)
    logits = torch.empty(5, 256, device="cuda")
    model.extend(cache, x[3:].contiguous(), [0, 5, 0], all_rows=True, logits=logits)
    assert [cache.length(r) for r in range(3)] == [0, 8, 0]
    close(logits, by_steps(sa, model, "f32", [x])[0][3:], "f32")
    assert model.extend(cache, x[:0].contiguous(), [0, 0, 0], all_rows=True).numel() == 0


@pytest.mark.parametrize("n", [3, 40])
def test_captured(sa, n):
    """A graph repeats the call for the lengths at the call, also after larger calls."""
    model = make_model(sa, 32, 400)
    cache = make_cache(sa, "bf16", 2, 400)
    model.extend(cache, tokens_of(200, 7).view(2, 100).contiguous())
    x = tokens_of(2 * n, 8).view(2, n).contiguous()
    want = torch.empty(2, 256, device="cuda")
    model.extend(cache, x, logits=want, commit=False)
    logits, new = torch.zeros_like(want), torch.zeros(2, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        model.extend(cache, x, logits=logits, next_tokens=new, commit=False)
    model.extend(cache, tokens_of(400, 9).view(2, 200).contiguous(), commit=False)     # larger
    for _ in range(3):
        logits.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(logits, want) and torch.equal(new.long(), want.argmax(-1))


def greedy(sa, model, kv, prompts, n, cfg=CFG):
    G, L = prompts.shape
    cache = make_cache(sa, kv, G, L + n, cfg)
    new = model.prefill(cache, prompts)
    out = [new]
    for _ in range(n - 1):
        new = model.decode_step(cache, new)
        out.append(new)
    return torch.stack(out, 1).tolist()


@pytest.mark.parametrize("drafter", ["itself", "another", "lookup"])
@pytest.mark.parametrize("n_draft", [0, 1, 4])
def test_greedy_speculation_equals_greedy_decoding(sa, drafter, n_draft):
    model = make_model(sa, 32, 200)
    prompts = tokens_of(3 * 20, 10).view(3, 20).contiguous()
    n = 33
    want = greedy(sa, model, "f32", prompts, n)
    draft = {"itself": model, "another": make_model(sa, 32, 200, seed=6), "lookup": None}[drafter]
    draft_cache = None if draft is None else make_cache(sa, "f32", 3, 60)
    got = model.speculative(make_cache(sa, "f32", 3, 60), prompts, n, draft, draft_cache, n_draft, temperature=0.0)
    assert got == want


def test_speculation_ends_at_eos(sa):
    model = make_model(sa, 32, 200)
    prompts = tokens_of(2 * 9, 11).view(2, 9).contiguous()
    want = greedy(sa, model, "f32", prompts, 20)
    eos = want[0][7]
    cut = [w[:w.index(eos) + 1] if eos in w else w for w in want]
    got = model.speculative(make_cache(sa, "f32", 2, 60), prompts, 20, model, make_cache(sa, "f32", 2, 60), 3, 0.0, eos=eos)
    assert got == cut


@pytest.mark.parametrize("kv", ["f32", "bf16", "fp8"])
def test_sampled_speculation(sa, kv):
    """Equal seeds give equal tokens; a draft model that is the model itself is mostly believed."""
    model = make_model(sa, 64, 200, CFG128)
    prompts = tokens_of(4 * 12, 12).view(4, 12).contiguous()
    runs = []
    for _ in range(2):
        gen = torch.Generator(device="cuda").manual_seed(1)
        runs.append(model.speculative(make_cache(sa, kv, 4, 64, CFG128), prompts, 25, model,
                                      make_cache(sa, kv, 4, 64, CFG128), 5, 0.9, generator=gen))
    assert runs[0] == runs[1]
    assert all(len(t) == 25 and all(0 <= x < 256 for x in t) for t in runs[0])


def test_refusals(sa):
    model = make_model(sa, 4, 100)
    cache = make_cache(sa, "f32", 2, 64)
    x = tokens_of(70, 13)
    with pytest.raises(sa.SaError, match="full"):
        model.extend(cache, x[:66].contiguous(), [65, 1])
    with pytest.raises(sa.SaError, match="RoPE"):
        model.extend(cache, tokens_of(102, 1), [101, 1])
    with pytest.raises(sa.SaError, match="new token"):
        model.extend(cache, x[:2].contiguous(), [2, 0])
    with pytest.raises(sa.SaError, match="new token"):
        model.extend(cache, x[:2].contiguous(), [3, -1], all_rows=True)
    with pytest.raises(sa.SaError, match="rows of logits"):
        model.extend(cache, x[:5].contiguous(), [3, 2], all_rows=True)
    with pytest.raises(sa.SaError, match="n_seq"):
        model.extend(cache, x[:3].contiguous(), [1, 1, 1])
    with pytest.raises(ValueError):
        model.extend(cache, x[:3].contiguous(), [1, 1])
    with pytest.raises(ValueError):
        model.extend(cache, x[:2].contiguous(), [1, 1], logits=torch.empty(2, 3, device="cuda"))
    other = make_cache(sa, "f32", 2, 64, CFG128)
    with pytest.raises(sa.SaError, match="geometry"):
        model.extend(other, x[:2].contiguous(), [1, 1])
    assert [cache.length(r) for r in range(2)] == [0, 0]
    p = tokens_of(8, 1).view(2, 4).contiguous()
    for bad in (dict(n_tokens=0), dict(n_draft=-1), dict(n_draft=65), dict(temperature=-1.0), dict(n_tokens=80),
                dict(n_draft=2), dict(draft=model)):
        with pytest.raises(ValueError):
            model.speculative(cache, p, **dict(dict(n_tokens=5, n_draft=1), **bad))
    fork = make_cache(sa, "f32", 2, 64)
    model.extend(fork, p[:1].contiguous())
    fork.set_len(0, 4)
    fork2 = sa.KVCache(2, 2, 64, 2, 1, 2)
    fork2.reserve(0, 64)
    fork2.set_len(0, 64)
    fork2.fork(1, 0, 64)
    fork2.set_lens([0, 1], [10, 10])          # back into a shared page
    with pytest.raises(sa.SaError, match="shares"):
        model.extend(fork2, x[:2].contiguous(), [1, 1])


def test_speculative_refuses_one_cache_for_both_models(sa):
    model = make_model(sa, 4, 100)
    cache = make_cache(sa, "f32", 2, 64)
    p = tokens_of(8, 1).view(2, 4).contiguous()
    with pytest.raises(ValueError, match="of its own"):
        model.speculative(cache, p, 5, draft=model, draft_cache=cache, n_draft=1)
    for bad in (p.long(), p[0], p.cpu()):
        with pytest.raises(ValueError, match="prompts"):
            model.speculative(cache, bad, 5, n_draft=1)
    assert [cache.length(r) for r in range(2)] == [0, 0]
