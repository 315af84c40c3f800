"""GPU tests of the verification where calls are large: whole segments inside rows, a wave
each (from 4096 segments of 2048 logits on), and rows of more segments than the
drawing workgroup has threads; against the definition in 64 bits, written apart
(numpy).

Results are whole numbers and have to be equal.  They could differ only where a
uniform number lies within the kernel's 1e-13 of a border (the sums here are taken in
more than 64 bits); the seeds are fixed.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

SEG = 2048     # logits of a segment


def probabilities(x, T):
    x = np.asarray(x, np.float64) / np.float64(np.float32(T))      # the call's temperature is a float
    top = np.max(x)
    if not np.isfinite(top):
        return None
    e = np.exp(x - top)
    return e / e.sum()


def draw(w, u):
    c = np.cumsum(w, dtype=np.longdouble)
    hit = int(np.searchsorted(c, np.longdouble(u) * c[-1], side="right"))
    return hit if hit < len(w) else int(np.nonzero(w > 0)[0][-1])


def greedy(x):
    x = np.where(np.isnan(x), -np.inf, x)
    return int(np.argmax(x)) if np.max(x) > -np.inf else -1


def want(target, draft, tokens, ua, us, counts, T):
    acc, out, row, first, width = [], [], 0, 0, max(counts) + 1
    for b, n in enumerate(counts):
        path = []
        while True:
            k = len(path)
            x, drafted = target[row + k], int(tokens[first + k]) if k < n else None
            if T == 0:
                token = greedy(x)
                if token < 0 or token != drafted:
                    break
            else:
                p, q, token = probabilities(x, T), None, -1
                if p is None:
                    break
                if drafted is not None:
                    if draft is None:
                        q = np.zeros(len(x))
                        q[drafted] = 1
                    else:
                        q = probabilities(draft[first + k], T)
                    if q is None or not float(ua[first + k]) * q[drafted] < p[drafted]:
                        w = p if q is None else np.maximum(p - q, 0)
                        token = draw(w if w.sum() > 0 else p, float(us[b]))
                        break
                    token = drafted
                else:
                    token = draw(p, float(us[b]))
                    break
            path.append(token)
        acc.append(len(path))
        out.append(path + [token] + [-1] * (width - len(path) - 1))
        row += n + 1
        first += n
    return acc, out


def inputs(V, counts, drafts, seed, agree=0.6):
    """A token of each drafted place stands out more or less; drafts are drawn, or are that token or any."""
    g = torch.Generator().manual_seed(seed)
    N, B = sum(counts), len(counts)
    target = torch.randn(N + B, V, generator=g) * 2.5
    at = torch.tensor([sum(counts[:b]) + b + k for b, n in enumerate(counts) for k in range(n)])
    fav = torch.randint(0, V, (N,), generator=g)
    target[at, fav] += 30 * torch.rand(N, generator=g)
    if drafts == "model":
        draft = target[at] + agree * torch.randn(N, V, generator=g)
        tokens = (draft - torch.log(-torch.log(torch.rand(N, V, generator=g).clamp(1e-7, 1 - 1e-7)))).argmax(-1)
    else:
        draft = None
        tokens = torch.where(torch.rand(N, generator=g) < 0.8, fav, torch.randint(0, V, (N,), generator=g))
    return target, draft, tokens.int(), torch.rand(N, generator=g), torch.rand(B, generator=g)


def on_gpu(t, offset, stride):
    """t on the GPU, its rows `stride` logits apart more than they are long, the first `offset` logits behind a 16-byte
    boundary; NaN between them."""
    rows, V = t.shape
    buf = torch.full((rows * (V + stride) + 8,), float("nan"), device="cuda")
    v = buf[offset:offset + rows * (V + stride)].view(rows, V + stride)[:, :V]
    v.copy_(t)
    return v


def compare(sa, x, counts, T, offset=0, stride=0):
    target, draft, tokens, ua, us = x
    exp = want(target.numpy(), None if draft is None else draft.numpy(), tokens.numpy(), ua.numpy(), us.numpy(), counts, T)
    got = sa.draft_verify(on_gpu(target, offset, stride), tokens.cuda(), ua.cuda(), us.cuda(), counts,
                          draft=None if draft is None else on_gpu(draft, 3 - offset, stride), temperature=T)
    assert (got[0].tolist(), got[1].tolist()) == exp
    return exp[0]


def segments(V, rows):
    return rows * -(-(V + 3) // SEG)


@pytest.mark.parametrize("drafts", ["model", "lookup"])
@pytest.mark.parametrize("offset,stride", [(0, 0), (0, 1), (1, 0), (2, 5), (3, 3)])
def test_many_whole_segments(sa, drafts, offset, stride):
    """64 sequences of 4 drafts; rows on every distance from a 16-byte boundary."""
    counts, V = [4] * 64, 32003
    assert segments(V, 320) >= 4096
    x = inputs(V, counts, drafts, 20 + offset)
    for T in (0.8, 0.0):
        acc = compare(sa, x, counts, T, offset, stride)
        assert set(acc) == {0, 1, 2, 3, 4}


@pytest.mark.parametrize("drafts", ["model", "lookup"])
def test_values_in_late_steps_of_a_segment(sa, drafts):
    """NaN, infinities, masked steps and logits far above all before them, anywhere in a wave's four steps."""
    counts, V = [4] * 64, 32003
    target, draft, tokens, ua, us = inputs(V, counts, drafts, 30)
    places = [0, 511, 512, 1023, 1024, 1535, 1536, 2000, 2047]
    for i in range(0, 320, 5):                       # the first place of each sequence: its first draft's
        at = 3 * SEG + places[(i // 5) % len(places)]
        kind = (i // 5) // len(places)
        if kind == 0:
            target[i, at] = float("nan")
        elif kind == 1:
            target[i, at] = 700.0                    # 2^1200 times the others' weight: the sum begins anew
        elif kind == 2:
            target[i, at], target[i, at + SEG - 900] = 3000.0, 5000.0
        elif kind == 3:
            target[i, 2 * SEG:at] = -float("inf")    # nothing before it in its segment
            target[i, at] = 60.0
        elif kind == 4:
            target[i, :at] = -float("inf")
        elif kind == 5:
            target[i, at:] = -float("inf")
        else:
            target[i, at] = float("inf")
    for k in range(0, 256, 4):                       # drafted tokens on the values that were put there
        b = k // 4
        if b % 2:
            tokens[k] = 3 * SEG + places[b % len(places)]
    if draft is not None:
        draft[1::8, 4 * SEG + 1600] = 900.0
        draft[5::16, 4 * SEG + 1700] = float("nan")
        draft[3::8, 5 * SEG:7 * SEG] = -float("inf")
    for T in (1.0, 0.7, 0.0):
        compare(sa, (target, draft, tokens, ua, us), counts, T)


@pytest.mark.parametrize("T", [1.0, 0.0])
def test_many_peaked_and_flat_rows(sa, T):
    """Logits of a spread of 1e4, a row of equal ones and ones of a spread of 1e-3."""
    counts, V = [4] * 64, 32003
    target, draft, tokens, ua, us = inputs(V, counts, "model", 31)
    for t in (target, draft):
        t[::4] *= 4e3
        t[1::4] = 1.25
        t[2::4] *= 4e-4
    at = torch.tensor([5 * b + k for b in range(64) for k in range(4)])     # target rows of the drafts
    tokens[::3] = target[at].argmax(-1).int()[::3]
    tokens[::4] = draft.argmax(-1).int()[::4]
    compare(sa, (target, draft, tokens, ua, us), counts, T)


@pytest.mark.parametrize("counts,drafts", [([2, 1, 0], "model"), ([1, 0], "model"), ([1, 1], "lookup"), ([3, 2, 0], "lookup")])
def test_more_segments_than_threads(sa, counts, drafts):
    """Rows of 587 segments; the uniform numbers reach to the last of them."""
    V = 1200001
    assert -(-(V + 3) // SEG) > 512
    for seed, u in ((40, None), (41, 1 - 2.0 ** -24), (42, 0.0)):
        x = list(inputs(V, counts, drafts, seed))
        if u is not None:
            x[4][:] = u
        for T in (1.0, 0.0):
            compare(sa, x, counts, T, 1, 2)


def test_sampling_many_rows(sa):
    n, V = 300, 30001
    assert segments(V, n) >= 4096
    g = torch.Generator().manual_seed(50)
    x, u = torch.randn(n, V, generator=g) * 2, torch.rand(n, generator=g)
    for T in (1.0, 0.2, 0.0):
        exp = [greedy(r) if T == 0 else draw(probabilities(r, T), float(w)) for r, w in zip(x.numpy(), u.numpy())]
        assert sa.sample(on_gpu(x, 2, 1), u.cuda(), temperature=T).tolist() == exp
