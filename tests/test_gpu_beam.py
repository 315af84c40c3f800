"""GPU tests of beam_select against log_softmax and a stable sort in 64 bits.

Tokens and beams have to be equal: candidates are ordered in 64 bits from
normalisers that are off by some 1e-8, and the inputs' candidates are further
apart or exactly equal.  Scores are rounded to fp32 (half a step, 2^-24
relative), beside a normaliser from fp32 sums of exponentials: each term is off
by at most 2^-22 of itself, so the logarithm by at most 2.4e-7."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def reference(logits, scores, n):
    """(scores, tokens, beams) in 64 bits on the host."""
    x, s = logits.double().cpu(), scores.double().cpu()
    G, B, V = x.shape
    lse = torch.logsumexp(x, -1)
    c = s[..., None] + x - lse[..., None]
    c = torch.where(torch.isfinite(lse)[..., None] & (c > -math.inf), c, -math.inf)
    c = torch.where(torch.isnan(c), -math.inf, c).reshape(G, -1)
    n_have = min(n, B * V)
    best, at = torch.sort(c, dim=-1, descending=True, stable=True)
    best, at = best[:, :n_have], at[:, :n_have]
    best = torch.nn.functional.pad(best, (0, n - n_have), value=-math.inf)
    at = torch.nn.functional.pad(at, (0, n - n_have), value=-1)
    none = best == -math.inf
    return best, torch.where(none, -1, at % V), torch.where(none, -1, at // V)


def check(sa, logits, scores, n):
    got = sa.beam_select(logits, scores, n)
    torch.cuda.synchronize()
    want = reference(logits, scores, n)
    assert torch.equal(got[1].cpu().long(), want[1]), (got[1], want[1])
    assert torch.equal(got[2].cpu().long(), want[2]), (got[2], want[2])
    a, b = got[0].cpu().double(), want[0]
    fine = b > -math.inf
    assert torch.equal(fine, a > -math.inf)
    assert ((a - b).abs()[fine] <= 2.4e-7 + 2.0 ** -24 * b.abs()[fine]).all(), (a - b).abs().max()


def inputs(G, B, V, seed, std=2.5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(G, B, V, device="cuda", generator=gen) * std,
            -20 * torch.rand(G, B, device="cuda", generator=gen))


@pytest.mark.parametrize("V", [1, 2, 7, 63, 64, 65, 511, 513, 1000, 4096, 32003, 151936])
@pytest.mark.parametrize("G,B,n", [(1, 1, 1), (1, 4, 8), (3, 5, 10), (2, 64, 64), (5, 3, 64)])
def test_sizes(sa, G, B, V, n):
    check(sa, *inputs(G, B, V, G * 1000 + B + V), n)


def test_long_rows(sa):
    """Segments of several steps."""
    check(sa, *inputs(1, 16, 1 << 20, 1), 32)
    check(sa, *inputs(2, 64, 151936, 2), 64)


@pytest.mark.parametrize("B,V,n", [(1, 5000, 16), (4, 151936, 8), (3, 130, 64), (8, 32003, 32)])
def test_equal_values(sa, B, V, n):
    """Ties go to the lowest index: all equal, a few levels, equal beams."""
    G = 2
    z = torch.zeros(G, B, V, device="cuda")
    s = torch.zeros(G, B, device="cuda")
    check(sa, z, s, n)
    gen = torch.Generator(device="cuda").manual_seed(V)
    check(sa, torch.randint(0, 3, (G, B, V), device="cuda", generator=gen).float(), s, n)
    x, _ = inputs(G, 1, V, 5)
    same = x.expand(G, B, V).contiguous()
    check(sa, same, s, n)
    # a lone best token behind many equal ones
    z[:, -1, V - 1] = 1.0
    check(sa, z, s, n)


def test_scores_far_from_the_logits(sa):
    """Accumulated scores so large that close logits make equal sums in 64 bits."""
    x, _ = inputs(1, 2, 3000, 6, std=1e-3)
    check(sa, x, torch.full((1, 2), -1e12, device="cuda"), 20)


@pytest.mark.parametrize("V", [40, 3000, 151936])
def test_masked_and_broken_rows(sa, V):
    G, B, n = 2, 6, 12
    x, s = inputs(G, B, V, 7)
    s[:, 1] = -math.inf                      # a beam not yet begun
    x[:, 2] = -math.inf                      # nothing possible
    x[0, 3, V // 2] = math.nan
    x[1, 3, V - 1] = math.inf
    s[0, 4] = math.nan
    x[:, 5, 3:] = -math.inf                  # three tokens left
    check(sa, x, s, n)
    x[:, 0] = -math.inf
    s[1, 4] = -math.inf
    check(sa, x, s, n)                       # fewer candidates than places
    x[:, 5] = -math.inf
    x[:, 4] = -math.inf
    check(sa, x, s, n)                       # none at all
    wild = torch.full((1, 2, V), -3.0e38, device="cuda")
    wild[0, 1, 5] = 3.0e38
    check(sa, wild, torch.zeros(1, 2, device="cuda"), 4)


def test_strided_rows(sa):
    buf = torch.randn(3, 4, 1030, device="cuda")
    s = torch.zeros(3, 4, device="cuda")
    check(sa, buf[:, :, 1:1004], s, 8)
    check(sa, buf[:, 2:3, 5:805][:, :1], s[:, :1].contiguous(), 8)
    with pytest.raises(ValueError):
        sa.beam_select(buf[:, 2:3], s[:, :1], 8)          # strided scores
    with pytest.raises(ValueError):
        sa.beam_select(buf[:, 1:3], s[:, :2], 4)          # uneven rows
    with pytest.raises(ValueError):
        sa.beam_select(buf[:, :, ::2], s, 4)
    with pytest.raises(ValueError):
        sa.beam_select(buf.double(), s, 4)
    with pytest.raises(ValueError):
        sa.beam_select(buf, s[:, :2], 4)


def test_refusals(sa):
    lib = sa.lib()
    x, s = inputs(1, 2, 100, 8)
    o = torch.full((64,), 7.0, device="cuda")
    i = torch.full((128,), 7, dtype=torch.int32, device="cuda")
    ws = torch.zeros(4096, dtype=torch.uint8, device="cuda")

    def call(x=x.data_ptr(), stride=100, s=s.data_ptr(), G=1, B=2, V=100, n=4, o=o.data_ptr(), ws=ws.data_ptr(), nb=4096):
        return lib.sa_beam_select(x, stride, s, G, B, V, n, o, i.data_ptr(), i.data_ptr() + 256, ws, nb, None)

    for bad in (dict(x=None), dict(s=None), dict(o=None), dict(G=0), dict(B=0), dict(B=65), dict(V=0), dict(n=0),
                dict(n=65), dict(stride=99), dict(ws=ws.data_ptr() + 4), dict(B=64, V=1 << 25, stride=1 << 25), dict(G=-1)):
        assert call(**bad) == sa.SA_EINVAL, bad
        assert lib.sa_last_error()
    assert call(nb=8) == sa.SA_ENOMEM and call(ws=None) == sa.SA_ENOMEM
    torch.cuda.synchronize()
    assert (o == 7).all() and (i == 7).all()
    assert call() == sa.SA_OK
    assert sa.beam_select_ws_bytes(1, 65, 10, 1) == 0 and sa.beam_select_ws_bytes(0, 1, 10, 1) == 0
    assert sa.beam_select_ws_bytes(1, 1, 10, 65) == 0 and sa.beam_select_ws_bytes(1, 4, 151936, 8) > 0


def test_graph_replays(sa):
    x, s = inputs(2, 4, 32003, 9)
    out = (torch.empty(2, 8, device="cuda"), *(torch.empty(2, 8, dtype=torch.int32, device="cuda") for _ in range(2)))
    ws = torch.empty(sa.beam_select_ws_bytes(2, 4, 32003, 8), dtype=torch.uint8, device="cuda")
    sa.beam_select(x, s, 8, out=out, ws=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sa.beam_select(x, s, 8, out=out, ws=ws)
    for rep in range(3):
        x.copy_(inputs(2, 4, 32003, 20 + rep)[0])
        ws.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        eager = sa.beam_select(x, s, 8)
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
        want = reference(x, s, 8)
        assert torch.equal(out[1].cpu().long(), want[1]) and torch.equal(out[2].cpu().long(), want[2])
    del graph


@pytest.mark.parametrize("B,V,n", [(8, 151936, 16), (16, 151936, 64), (33, 70001, 64)])
def test_equal_values_in_eight_segments_a_thread(sa, B, V, n):
    z = torch.zeros(1, B, V, device="cuda")
    s = torch.zeros(1, B, device="cuda")
    check(sa, z, s, n)
    gen = torch.Generator(device="cuda").manual_seed(V + B)
    check(sa, torch.randint(0, 3, (1, B, V), device="cuda", generator=gen).float(), s, n)
    z[:, -1, V - 1] = 1.0
    check(sa, z, s, n)


@pytest.mark.parametrize("B", [1, 4, 8, 16])
def test_few_tokens_allowed(sa, B):
    """A mask that leaves a few tokens of a long vocabulary: most segments, and
    whole waves of them, hold nothing but -inf, one of them a NaN beside it."""
    V = 151936
    x, s = inputs(2, B, V, 60 + B)
    allowed = torch.tensor([3, 70000, 70001, V - 1], device="cuda")
    masked = torch.full_like(x, -math.inf)
    masked[..., allowed] = x[..., allowed]
    check(sa, masked, s, 8)
    masked[1, B - 1, 40000] = math.nan
    check(sa, masked, s, 8)


def test_sums_of_many_steps(sa):
    """Segments of 128 steps alike, whose sums would round the same way again and
    again.  Scores that take the normaliser away leave its error: the exponential's
    argument below 1.5 (half a step, 4.2e-8 of the value) and result (2^-23), sums of
    eight equal values (the four that are not exact round by at most (3 + 5 + 6 + 7) /
    8 x 2^-24) and of lanes of which one differs (1 + 1/2 + .. + 1/32 x 2^-24), the
    segment's sum to fp32 (2^-24) and its factor exp(-0.01) (result 2^-23, product
    2^-24): 6.8e-7."""
    B, V = 64, 1 << 23
    u = torch.linspace(0.3, 1.0, B, dtype=torch.float32)
    x = torch.empty(1, B, V, device="cuda")
    x[0] = -u.cuda()[:, None]
    x[0, :, ::512] = 0
    x[0, :, 0] = 0.01
    most = x[0, 0, 0].double().item()
    lse = torch.log(math.exp(most) + (V // 512 - 1) + (V - V // 512) * torch.exp(-u.double()))
    scores = lse.float()
    c, t, b = sa.beam_select(x, scores.cuda()[None], B)
    assert (t == 0).all() and sorted(b[0].tolist()) == list(range(B))
    want = (most + scores.double() - lse)[b[0].cpu().long()]
    assert (c[0].cpu().double() - want).abs().max().item() <= 6.8e-7 + 2.0 ** -24 * 0.02


@pytest.mark.parametrize("B,V", [(64, 300001), (64, 4500000), (33, 1000003)])
def test_steps_that_rise(sa, B, V):
    """Every step of a segment has a larger maximum than those before it, or a
    smaller one."""
    gen = torch.Generator(device="cuda").manual_seed(V)
    x = torch.randn(1, B, V, device="cuda", generator=gen) * 0.1 + torch.linspace(0, 5, V, device="cuda")
    s = -torch.rand(1, B, device="cuda", generator=gen)
    for logits in (x, x.flip(-1).contiguous()):
        c, t, b = sa.beam_select(logits, s, 16)
        lp = torch.log_softmax(logits[0].double(), -1) + s[0].double()[:, None]
        best, at = torch.topk(lp.view(-1), 16)
        assert torch.equal(b[0].long() * V + t[0].long(), at)
        assert ((c[0].double() - best).abs() <= 2.4e-7 + 2.0 ** -24 * best.abs()).all()
