"""GPU tests of what speculative generation promises beyond equal greedy tokens: a model
that drafts for itself is believed, tokens are distributed as the target's own
whatever drafts them, what cannot run is refused before it begins, and logits
without a distribution end a generation with an error."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_speculative import CFG128, greedy, make_cache, make_model, tokens_of

pytestmark = pytest.mark.gpu


@pytest.fixture
def rounds(sa, monkeypatch):
    """(drafted, accepted) tokens of each sequence in every verification of a generation."""
    seen, verify = [], sa.draft_verify

    def record(target, tokens, u_accept, u_sample, counts, **k):
        out = verify(target, tokens, u_accept, u_sample, counts, **k)
        seen.append((list(counts), out[0].tolist()))
        return out
    monkeypatch.setattr(sa, "draft_verify", record)
    return seen


@pytest.mark.parametrize("T", [0.9, 0.3])
def test_a_model_believes_itself(sa, rounds, T):
    """fp32 caches: p and q are equal but for the order of sums, so that all drafts are accepted (one is rejected with
    a probability of |p / q - 1|, some 1e-5)."""
    G, n, n_draft = 4, 25, 5
    model = make_model(sa, 64, 200, CFG128)
    prompts = tokens_of(G * 12, 12).view(G, 12).contiguous()
    gen = torch.Generator(device="cuda").manual_seed(2)
    got = model.speculative(make_cache(sa, "f32", G, 64, CFG128), prompts, n, model, make_cache(sa, "f32", G, 64, CFG128),
                            n_draft, T, generator=gen)
    assert [len(t) for t in got] == [n] * G
    drafted = [r for r in rounds if sum(r[0])]
    assert all(counts == accepted for counts, accepted in drafted)
    assert len(drafted) == math.ceil((n - 1) / (n_draft + 1))


def conditional(model, sa, prompts, texts, T):
    """The target's probabilities of every token of texts [G, n] behind its prompt and the ones before it, in 64 bits."""
    G, n = texts.shape
    cache = make_cache(sa, "f32", G, prompts.shape[1] + n, CFG128)
    logits = torch.empty(G, CFG128["vocab"], device="cuda")
    model.prefill(cache, prompts, logits=logits)
    out = []
    for i in range(n):
        out.append(torch.softmax(logits.double() / T, -1))
        model.decode_step(cache, texts[:, i].contiguous(), logits=logits)
    return torch.stack(out, 1)


def similar(sa, max_batch):
    """make_model's model with another final norm."""
    model = make_model(sa, max_batch, 64, CFG128)
    norm = model.tensor(sa.QW_FINAL_NORM)
    norm.mul_(1 + 0.5 * torch.randn(norm.numel(), generator=torch.Generator().manual_seed(4)).cuda())
    return model


@pytest.mark.parametrize("drafter", ["similar", "lookup"])
def test_tokens_are_distributed_as_the_targets(sa, rounds, drafter):
    """Given what stands before it, each token is drawn from the target's softmax: for any f of a token and its past, the
    sum of f minus its mean under p is one of terms of mean 0, normal in the limit.  5.5 standard deviations
    are exceeded with a probability of 4e-8 by each of the 265 sums; rare tokens' sums are not yet normal, and
    Bernstein's inequality bounds theirs by sqrt(2 V x) + 2 x / 3 at exp(-x), x = 5.5^2 / 2."""
    G, n, n_draft, T = 128, 12, 3, {"similar": 0.8, "lookup": 0.25}[drafter]
    model = make_model(sa, G * (n_draft + 1), 64, CFG128)
    draft = similar(sa, G * (n_draft + 1)) if drafter == "similar" else None
    gen = torch.Generator(device="cuda").manual_seed(3)
    dev = var = 0.0
    for run in range(6):
        start = tokens_of(G * 4, 60 + run).view(G, 4)
        prompts = torch.cat([start, start, start[:, :2]], 1).contiguous()        # something to look up
        caches = [make_cache(sa, "f32", G, 64, CFG128) for _ in range(2)]
        got = model.speculative(caches[0], prompts, n, draft, None if draft is None else caches[1], n_draft, T, generator=gen)
        texts = torch.tensor(got, dtype=torch.int32, device="cuda")
        p = conditional(model, sa, prompts, texts, T)                             # [G, n, V]
        hit = torch.zeros_like(p).scatter_(2, texts.long()[..., None], 1.0)
        logp = p.clamp_min(1e-300).log()
        # what a draft model prefers shows what it drafts and is not rejected as often as it should be
        other = p if draft is None else conditional(draft, sa, prompts, texts, T)
        tests = [logp.clamp_min(-30.0), (logp - other.clamp_min(1e-300).log()).clamp(-30.0, 30.0), p,
                 (p > p.amax(-1, keepdim=True) / 4).double()]
        before = torch.cat([prompts[:, -1:], texts[:, :-1]], 1).long()[..., None]
        tokens = torch.arange(p.shape[-1], device="cuda")
        tests += [((tokens + before) % m < m / 2).double() for m in (2, 3, 5, 16, 64)]
        for f in (torch.stack(tests), None):
            if f is None:      # every token's own indicator
                d, v = (hit - p).sum((0, 1)), (p * (1 - p)).sum((0, 1))
            else:
                mean = (f * p).sum(-1)
                d, v = ((f * hit).sum(-1) - mean).sum((1, 2)), ((f * f * p).sum(-1) - mean ** 2).sum((1, 2))
            sums = (d, v) if f is not None else (torch.cat([sums[0], d]), torch.cat([sums[1], v]))
        dev, var = dev + sums[0], var + sums[1]
    x = 5.5 ** 2 / 2
    wide = torch.ones_like(dev)
    wide[0], wide[1] = 30.0, 60.0             # the largest |f - E f|
    assert (dev.abs() <= (2 * var * x).sqrt() + 2 * x / 3 * wide).all(), (dev / var.sqrt())[:9].tolist()
    drafted, accepted = (sum(sum(r[i]) for r in rounds) for i in (0, 1))
    assert 0.1 * drafted < accepted < 0.9 * drafted and drafted > G * 6, (drafted, accepted)


@pytest.mark.parametrize("n_tokens", [1, 5])
@pytest.mark.parametrize("T", [1.0, 0.0])
def test_logits_without_a_distribution(sa, n_tokens, T):
    """The prompt's own logits are looked at as later ones are."""
    model = make_model(sa, 16, 100)
    model.tensor(sa.QW_FINAL_NORM).fill_(float("nan"))
    p = tokens_of(8, 1).view(2, 4).contiguous()
    with pytest.raises(ValueError, match="distribution"):
        model.speculative(make_cache(sa, "f32", 2, 64), p, n_tokens, n_draft=2, temperature=T)


@pytest.mark.parametrize("drafter", ["itself", "lookup"])
@pytest.mark.parametrize("n_draft", [0, 1, 3, 6])
def test_what_follows_eos_does_not_matter(sa, drafter, n_draft):
    """Logits behind an accepted eos are no token's, whatever they are."""
    model = make_model(sa, 32, 200)
    prompts = tokens_of(2 * 9, 11).view(2, 9).contiguous()
    want = greedy(sa, model, "f32", prompts, 20)
    eos = want[0][7]
    assert not (prompts == eos).any()
    model.tensor(sa.QW_EMBED).view(256, -1)[eos] = float("nan")
    draft, caches = (model if drafter == "itself" else None), [make_cache(sa, "f32", 2, 60) for _ in range(2)]
    got = model.speculative(caches[0], prompts, 20, draft, None if draft is None else caches[1], n_draft, 0.0, eos=eos)
    assert got == [w[:w.index(eos) + 1] if eos in w else w for w in want]


def test_refused_before_it_begins(sa):
    """Neither cache has changed where either does not fit."""
    model, short = make_model(sa, 16, 100), make_model(sa, 16, 10)
    p = tokens_of(8, 1).view(2, 4).contiguous()
    new = lambda pages=2, cfg=None: sa.KVCache(2, 2, 64 if cfg is None else cfg["head_dim"], 2, pages, 2 * pages)  # noqa: E731

    def refused(draft, draft_cache, match, cache=None):
        cache = new() if cache is None else cache
        before = [[(c.length(r), c.capacity(r)) for r in range(2)] for c in (cache, draft_cache)]
        with pytest.raises(ValueError, match=match):
            model.speculative(cache, p, 20, draft=draft, draft_cache=draft_cache, n_draft=2)
        assert [[(c.length(r), c.capacity(r)) for r in range(2)] for c in (cache, draft_cache)] == before

    refused(short, new(), "positions")
    refused(make_model(sa, 2, 100), new(), "row per sequence")
    used = new()
    used.reserve(1, 64)
    used.set_len(1, 3)
    refused(model, used, "empty")
    refused(model, new(), "empty", cache=used)
    refused(model, new(cfg=CFG128), "geometry")
    refused(model, new(), "geometry", cache=new(cfg=CFG128))
