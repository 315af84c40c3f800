"""GPU tests of the verification of drafted tokens and of sampling, against the
definition in 64 bits, written apart (numpy).

Results are whole numbers and have to be equal.  They could differ only where a
uniform number lies within the kernel's 1e-13 of a border; the seeds are fixed.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def softmax(x, T):
    x = np.asarray(x, np.float64) / T
    top = np.max(x) if len(x) else -np.inf
    if not np.isfinite(top):
        return None
    e = np.exp(x - top)
    s = e.sum()
    return e / s if np.isfinite(s) and s > 0 else None


def draw(w, u):
    c = np.cumsum(w)
    hit = np.nonzero(c > u * c[-1])[0]
    return int(hit[0]) if len(hit) else int(np.nonzero(w > 0)[0][-1])


def want(target, draft, tokens, ua, us, counts, T, width):
    acc, out, row, first = [], [], 0, 0
    V = target.shape[1]
    for b, n in enumerate(counts):
        path, token = [], -1
        for k in range(n + 1):
            x = target[row + k]
            if T == 0:
                ok = ~np.isnan(x) & (x > -np.inf)
                best = int(np.argmax(np.where(ok, x, -np.inf))) if ok.any() else -1
                if k < n and best >= 0 and tokens[first + k] == best:
                    path.append(best)
                    continue
                token = best
                break
            p = softmax(x, T)
            q = None
            if k < n:
                t = int(tokens[first + k])
                if draft is None:
                    q = np.zeros(V)
                    if 0 <= t < V:
                        q[t] = 1
                else:
                    q = softmax(draft[first + k], T)
                if p is not None and q is not None and 0 <= t < V and float(ua[first + k]) * q[t] < p[t]:
                    path.append(t)
                    continue
            if p is not None:
                w = p if q is None else np.maximum(p - q, 0)
                token = draw(w if w.sum() > 0 else p, float(us[b]))
            break
        acc.append(len(path))
        out.append(path + [token] + [-1] * (width - len(path) - 1))
        row += n + 1
        first += n
    return acc, out


def inputs(V, counts, drafts, seed, spread=2.5, agree=0.6):
    g = torch.Generator().manual_seed(seed)
    N, B = sum(counts), len(counts)
    target = torch.randn(N + B, V, generator=g) * spread
    at = [sum(counts[:b]) + b + k for b, n in enumerate(counts) for k in range(n)]
    if drafts == "model":
        draft = target[at] + agree * torch.randn(N, V, generator=g)
        tokens = torch.multinomial(torch.softmax(draft, -1), 1, generator=g)[:, 0] if N else torch.zeros(0)
    else:
        draft = None
        tokens = target[at].argmax(-1) if N else torch.zeros(0)
        tokens = torch.where(torch.rand(N, generator=g) < 0.3, torch.randint(0, V, (N,), generator=g), tokens.long())
    return target, draft, tokens.int(), torch.rand(N, generator=g), torch.rand(B, generator=g)


def run(sa, target, draft, tokens, ua, us, counts, T):
    acc, out = sa.draft_verify(target.cuda(), tokens.cuda(), ua.cuda(), us.cuda(), counts,
                               draft=None if draft is None else draft.cuda(), temperature=T)
    return acc.tolist(), out.tolist()


def compare(sa, x, counts, T):
    target, draft, tokens, ua, us = x
    exp = want(target.numpy(), None if draft is None else draft.numpy(), tokens.numpy(), ua.numpy(), us.numpy(), counts, T,
               max(counts) + 1)
    assert run(sa, *x, counts, T) == exp
    return exp


@pytest.mark.parametrize("drafts", ["model", "lookup"])
@pytest.mark.parametrize("V", [1, 2, 3, 5, 63, 64, 1023, 1024, 1025, 4097, 32003])
def test_vocabularies(sa, V, drafts):
    counts = [3, 0, 1, 5]
    for T in (1.0, 0.3, 2.0, 0.0):
        compare(sa, inputs(V, counts, drafts, V), counts, T)


@pytest.mark.parametrize("drafts", ["model", "lookup"])
def test_the_decoders_vocabulary(sa, drafts):
    counts = [4, 2, 0, 7, 1]
    acc = [compare(sa, inputs(151936, counts, drafts, seed), counts, 0.8)[0] for seed in (1, 2)]
    if drafts == "model":
        assert any(a not in (0, n) for row in acc for a, n in zip(row, counts))   # some are cut in the middle


def test_many_sequences_and_drafts(sa):
    """More sequences than a launch takes; up to 64 drafts, all of them accepted in some."""
    counts = [64, 0, 63, 1] + [i % 6 for i in range(140)]
    x = list(inputs(300, counts, "model", 5, agree=0.02))
    x[3][:64] = 0.0
    acc, _ = compare(sa, x, counts, 1.0)
    assert acc[0] == 64


def test_flat_and_peaked_rows(sa):
    counts = [2, 2, 2]
    for spread in (0.0, 1e-3, 30.0, 1e4):
        compare(sa, inputs(5000, counts, "model", 6, spread=spread), counts, 1.0)
    compare(sa, inputs(5000, counts, "lookup", 6, spread=1e4), counts, 1e-3)
    compare(sa, inputs(5000, counts, "model", 6), counts, 1e4)


def test_masked_tokens(sa):
    counts = [3, 3, 0]
    target, draft, tokens, ua, us = inputs(2500, counts, "model", 7)
    target[:, 5:2400] = -float("inf")
    draft[::2, 100:] = -float("inf")
    target[2, :] = -float("inf")
    target[2, 1234] = 3.0
    x = (target, draft, tokens, ua, us)
    for T in (1.0, 0.0):
        compare(sa, x, counts, T)
    lowest = target.clone()
    lowest[lowest == -float("inf")] = torch.finfo(torch.float32).min
    compare(sa, (lowest, draft, tokens, ua, us), counts, 1.0)


def test_rows_without_a_distribution(sa):
    counts = [2, 2, 2, 2, 2, 0]
    target, draft, tokens, ua, us = inputs(1500, counts, "model", 8)
    ua[:] = 0.0                                # all would be accepted
    target[1, 7] = float("nan")
    target[3] = -float("inf")
    draft[4, 1100] = float("nan")
    draft[6] = -float("inf")
    target[13, 3] = float("inf")
    target[15, 1400] = float("nan")
    x = (target, draft, tokens, ua, us)
    acc, out = compare(sa, x, counts, 1.0)
    assert acc == [1, 0, 0, 0, 1, 0] and out[0][1] == -1 and out[1][0] == -1 and out[2][0] >= 0 and out[5][0] == -1
    compare(sa, x, counts, 0.0)


def test_drafted_tokens_outside_the_vocabulary(sa):
    counts = [2, 1, 1]
    for drafts in ("model", "lookup"):
        target, draft, tokens, ua, us = inputs(100, counts, drafts, 9)
        tokens[0], tokens[2], tokens[3] = -1, 100, 2 ** 31 - 1
        ua[:] = 0.0
        x = (target, draft, tokens, ua, us)
        assert run(sa, *x, counts, 1.0)[0] == [0, 0, 0]
        compare(sa, x, counts, 1.0)
        assert run(sa, *x, counts, 0.0)[0] == [0, 0, 0]


def test_equal_logits_and_borders(sa):
    """Ties go to the lowest token; a uniform number on a border to the token behind it."""
    V = 4096
    target = torch.zeros(5, V)
    u = torch.tensor([0.0, 0.25, 0.5, 1 / V, 1 - 2.0 ** -24])
    none = torch.zeros(0)
    got = sa.sample(target.cuda(), u.cuda())
    assert got.tolist() == [0, V // 4, V // 2, 1, V - 1]
    assert sa.sample(target.cuda(), u.cuda(), temperature=0.0).tolist() == [0] * 5
    target[:, 9] = 1.0
    target[:, 2000] = 1.0
    assert sa.sample(target.cuda(), u.cuda(), temperature=0.0).tolist() == [9] * 5
    assert none.numel() == 0


def test_equal_distributions_accept_all(sa):
    """p = q: every draft is accepted whatever u < 1 is."""
    counts = [5, 5]
    target, _, _, _, us = inputs(3000, counts, "model", 10)
    draft = target[[0, 1, 2, 3, 4, 6, 7, 8, 9, 10]].clone()
    tokens = draft.argmax(-1).int()
    ua = torch.full((10,), 1 - 2.0 ** -24)
    assert run(sa, target, draft, tokens, ua, us, counts, 0.7)[0] == [5, 5]


def test_samples_are_distributed_as_the_target(sa):
    """Over an even grid of uniform numbers, first tokens fall as often as p says, whatever the draft."""
    V, A, S = 7, 64, 64
    g = torch.Generator().manual_seed(11)
    t, d = torch.randn(V, generator=g), torch.randn(V, generator=g)
    p, q = torch.softmax(t.double(), 0), torch.softmax(d.double(), 0)
    n = V * A * S
    grid = torch.cartesian_prod(torch.arange(V), torch.arange(A), torch.arange(S))
    acc, out = sa.draft_verify(t.expand(2 * n, V).contiguous().cuda(), grid[:, 0].int().cuda(),
                               ((grid[:, 1] + 0.5) / A).float().cuda(), ((grid[:, 2] + 0.5) / S).float().cuda(), [1] * n,
                               draft=d.expand(n, V).contiguous().cuda())
    weight = (q / (A * S))[grid[:, 0]]
    freq = torch.zeros(V, dtype=torch.float64).scatter_add_(0, out[:, 0].cpu().long(), weight)
    assert (freq - p).abs().max().item() <= 1.0 / A + 1.0 / S
    rate = (weight * acc.cpu()).sum().item()
    assert abs(rate - torch.minimum(p, q).sum().item()) <= V / 2 / A


@pytest.mark.parametrize("offset,stride", [(0, 0), (1, 0), (2, 5), (3, 1), (1, 2)])
def test_strided_and_unaligned_rows(sa, offset, stride):
    counts, V = [3, 1, 0, 2], 2051
    x = inputs(V, counts, "model", 12)
    exp = want(x[0].numpy(), x[1].numpy(), *[t.numpy() for t in x[2:]], counts, 1.0, 4)
    views = []
    for t, o in ((x[0], offset), (x[1], 3 - offset)):
        buf = torch.full((t.shape[0] * (V + stride) + 8,), float("nan"), device="cuda")
        v = buf[o:o + t.shape[0] * (V + stride)].view(t.shape[0], V + stride)[:, :V]
        v.copy_(t)
        views.append(v)
    acc, out = sa.draft_verify(views[0], x[2].cuda(), x[3].cuda(), x[4].cuda(), counts, draft=views[1])
    assert (acc.tolist(), out.tolist()) == exp


@pytest.mark.parametrize("T", [0.9, 0.0])
def test_captured_and_on_another_stream(sa, T):
    counts, V = [3, 4], 20000
    x = [t.cuda() for t in inputs(V, counts, "model", 13)]
    call = lambda **k: sa.draft_verify(x[0], x[2], x[3], x[4], counts, draft=x[1], temperature=T, **k)  # noqa: E731
    first = [t.clone() for t in call()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = call(stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, first))
    out = [torch.zeros_like(t) for t in first]
    ws = torch.empty(sa.draft_verify_ws_bytes(counts, V), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out=tuple(out), ws=ws)
    for _ in range(3):
        x[4].copy_(torch.rand(2))
        x[0].add_(torch.randn(V, device="cuda") * 0.5)
        ws.fill_(255)
        now = call()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, now))


def test_outputs_wider_than_needed(sa):
    """out_stride above what the counts need: -1 behind the drawn token."""
    import ctypes as C
    counts, V = [1, 0], 50
    target, _, tokens, ua, us = (None if t is None else t.cuda() for t in inputs(V, counts, "lookup", 14))
    acc = torch.zeros(2, dtype=torch.int32, device="cuda")
    out = torch.full((3, 5), 77, dtype=torch.int32, device="cuda")
    ws = torch.empty(sa.draft_verify_ws_bytes(counts, V), dtype=torch.uint8, device="cuda")
    arr = (C.c_int32 * 2)(*counts)
    sa.check(sa.lib().sa_draft_verify(target.data_ptr(), V, None, 0, tokens.data_ptr(), ua.data_ptr(), us.data_ptr(), 2, arr,
                                      V, 1.0, acc.data_ptr(), out.data_ptr(), 5, ws.data_ptr(), ws.numel(), None))
    torch.cuda.synchronize()
    rows = out.tolist()
    assert rows[2] == [77] * 5 and rows[1][1:] == [-1] * 4 and rows[1][0] >= 0 and rows[0][2:] == [-1] * 3


def test_sample_arguments(sa):
    x = torch.zeros(2, 5, device="cuda")
    u = torch.zeros(2, device="cuda")
    with pytest.raises(ValueError):
        sa.sample(x.double(), u)
    with pytest.raises(ValueError):
        sa.sample(x, u[:1])
    with pytest.raises(ValueError):
        sa.sample(x.t(), u)
    with pytest.raises(ValueError):
        sa.sample(x, u, out=torch.zeros(2, device="cuda"))
    with pytest.raises(sa.SaError, match="temperature"):
        sa.sample(x, u, temperature=-1.0)
    with pytest.raises(ValueError):
        sa.draft_verify(x, u.int(), u, u[:1], [1])          # a token per draft
