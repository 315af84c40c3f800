"""GPU tests of single-token attention over ranges of a paged cache: the
windowed decode (sliding window and sinks) and the decode of rows that share
their leading pages, against softmax(scale q k^T) v in 64 bits over the tokens
each row sees.

Tolerance: a score is a sum of 128 products of three-term operands, off by at
most about 131 x 2^-24 of sum |q_d k_d| scale, 7 for N(0,1) inputs: 5.6e-5; an
output of weights that are off by twice that, over values of mean 0.8, by
9e-5.  max-abs 1e-4 is therefore the bound, as in the other fp32 attention
tests; errors of random sign come out far smaller, relative L2 at most 2e-6.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


class Rows:
    """A cache on shuffled pages whose unwritten places hold NaN, and its rows'
    keys and values as they are stored."""

    def __init__(self, sa, kv, Hkv, D, lens, seed, spare=2, layers=1, width=1):
        self.sa, self.Hkv, self.D = sa, Hkv, D
        self.dtype = torch.bfloat16 if kv == "bf16" else torch.float32
        counts = [(n + 64) // 64 for n in lens]
        pages = sum(counts) + spare
        self.cache = sa.KVCache(layers, Hkv, D, len(lens), max(width, *counts, 0), pages,
                                sa.SA_DTYPE_BF16 if kv == "bf16" else sa.SA_DTYPE_F32)
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        for layer in range(layers):
            for view in sa.kv_pool_views(self.cache, layer):
                view.fill_(float("nan"))
        perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        self.k, self.v = [], []
        at = 0
        for r, (n, c) in enumerate(zip(lens, counts)):
            self.cache.set_pages(r, perm[at:at + c])
            at += c
            self.k.append(torch.empty(0, Hkv, D, device="cuda"))
            self.v.append(torch.empty(0, Hkv, D, device="cuda"))
            self.append(r, n)

    def append(self, r, n, commit=True, scale=1.0):
        if n == 0:
            return
        k, v = (torch.randn(n, self.Hkv, self.D, device="cuda", generator=self.gen) * scale for _ in range(2))
        self.cache.append(0, None, k[None], v[None], seq_ids=[r])
        if commit:
            self.cache.commit(n, seqs=[r])
        self.k[r] = torch.cat([self.k[r], k.to(self.dtype).float()])
        self.v[r] = torch.cat([self.v[r], v.to(self.dtype).float()])

    def fork(self, dst, src, n):
        self.cache.fork(dst, src, n)
        self.k[dst], self.v[dst] = self.k[src][:n], self.v[src][:n]

    def want(self, q, ids, scale, window=1 << 30, sink=0, drop=0):
        out = []
        for i, r in enumerate(ids):
            n = self.k[r].shape[0] - drop
            t = torch.arange(n, device="cuda")
            t = t[(n - 1 - t < window) | (t < sink)]
            if not n:
                out.append(torch.zeros_like(q[i], dtype=torch.float64))
                continue
            rep = q.shape[1] // self.Hkv
            k, v = (x[r][t].double().repeat_interleave(rep, 1) for x in (self.k, self.v))
            w = torch.softmax((q[i].double()[None] * k).sum(-1) * scale, 0)       # [T, Hq]
            out.append((w[..., None] * v).sum(0))
        return torch.stack(out)

    def query(self, n, rep):
        return torch.randn(n, self.Hkv * rep, self.D, device="cuda", generator=self.gen)


def close(got, want, rel=2e-6):
    assert torch.isfinite(got).all()
    err = (got.double() - want).abs().max().item()
    assert err <= 1e-4, err
    norm = want.norm().item()
    assert (got.double() - want).norm().item() <= rel * max(norm, 1e-30), (got.double() - want).norm().item() / norm


LENS = [0, 1, 31, 32, 33, 63, 64, 65, 100, 127, 128, 200, 500]


@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hkv,rep", [(2, 2), (1, 1), (3, 8), (1, 24), (2, 64)])
def test_window_heads(sa, kv, D, Hkv, rep):
    r = Rows(sa, kv, Hkv, D, LENS, 1)
    q = r.query(len(LENS), rep)
    for window, sink in ((100, 4), (64, 0), (1, 1)):
        got = r.cache.decode_window(0, q, D ** -0.5, window, sink)
        close(got, r.want(q, range(len(LENS)), D ** -0.5, window, sink))
    r.cache.close()


@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("window", [1, 31, 32, 33, 64, 90, 499, 500, 501, 2 ** 31 - 1])
@pytest.mark.parametrize("sink", [0, 1, 5, 32, 64, 70, 410, 2 ** 31 - 1])
def test_window_edges(sa, kv, window, sink):
    r = Rows(sa, kv, 2, 64, LENS, 2)
    q = r.query(len(LENS), 2)
    got = r.cache.decode_window(0, q, 0.125, window, sink)
    close(got, r.want(q, range(len(LENS)), 0.125, window, sink))
    r.cache.close()


@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("kv_block", [0, 64, 128, 1024])
def test_window_chunks(sa, kv, kv_block):
    """Long contexts in many chunks and in few; rows in any order and twice; a pending token."""
    lens = [5000, 3, 777, 2048]
    r = Rows(sa, kv, 2, 128, lens, 3)
    ids = [2, 0, 0, 3, 1]
    q = r.query(len(ids), 4)
    sa.set_attention_blocks(0, kv_block)
    try:
        got = r.cache.decode_window(0, q, 0.1, 3000, 70, seq_ids=ids)
        close(got, r.want(q, ids, 0.1, 3000, 70))
        for row in range(4):
            r.append(row, 1, commit=False)
        got = r.cache.decode_window(0, q, -0.1, 1000, 4, n_pending=1, seq_ids=ids)     # a negative scale
        close(got, r.want(q, ids, -0.1, 1000, 4))
        got = r.cache.decode_window(0, q, 0.1, 1000, 4, seq_ids=ids)                   # the token not yet counted
        close(got, r.want(q, ids, 0.1, 1000, 4, drop=1))
    finally:
        sa.set_attention_blocks(0, 0)
    r.cache.close()


@pytest.mark.parametrize("kv", ["f32", "bf16"])
def test_window_hidden_places_do_not_matter(sa, kv):
    """NaN and infinities in the keys and values that a row does not see."""
    n, window, sink = 700, 150, 10
    r = Rows(sa, kv, 2, 64, [n], 4)
    q = r.query(1, 2)
    first = r.cache.decode_window(0, q, 0.125, window, sink)
    want = r.want(q, [0], 0.125, window, sink)
    close(first, want)
    for bad in (float("nan"), float("inf"), -float("inf")):
        k, v = r.k[0].clone(), r.v[0].clone()
        k[sink:n - window], v[sink:n - window] = bad, bad
        r.cache.set_len(0, 0)
        r.cache.append(0, None, k[None], v[None], seq_ids=[0])
        r.cache.commit(n, seqs=[0])
        assert torch.equal(r.cache.decode_window(0, q, 0.125, window, sink), first)
    r.cache.close()


@pytest.mark.parametrize("kv", ["f32", "bf16"])
def test_large_scores(sa, kv):
    """Scores of hundreds, growing along the row: the running max is raised often."""
    r = Rows(sa, kv, 1, 128, [0], 5, spare=12, width=10)
    r.cache.reserve(0, 600)
    for i in range(12):
        r.append(0, 50, scale=2.0 + i)
    q = r.query(1, 4)
    for window in (1000, 90):
        want = r.want(q, [0], 1.0, window, 3)
        got = r.cache.decode_window(0, q, 1.0, window, 3)
        # scores of up to 13 x 128: their rounding, 131 x 2^-24 x 1500, moves a weight by 1e-2 at most
        err = (got.double() - want).norm().item() / want.norm().item()
        assert torch.isfinite(got).all() and err <= 1e-2, err
    r.cache.close()


def shared_rows(sa, kv, Hkv, D, prompts, tails, seed):
    """Groups of rows forked off prompts, each with a tail of its own."""
    lens, firsts = [], []
    for p, t in zip(prompts, tails):
        firsts.append(len(lens))
        lens += [p] + [0] * (len(t) - 1)
    total = sum((p + max(t)) // 64 + 2 + len(t) * (max(t) // 64 + 2) for p, t in zip(prompts, tails))
    r = Rows(sa, kv, Hkv, D, lens, seed, spare=total, width=max(p + max(t) for p, t in zip(prompts, tails)) // 64 + 2)
    for f, p, t in zip(firsts, prompts, tails):
        for i in range(1, len(t)):
            r.fork(f + i, f, p)
        for i, n in enumerate(t):
            r.cache.reserve(f + i, p + n)
            r.append(f + i, n)
    return r, [len(t) for t in tails]


@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hkv,rep", [(2, 2), (1, 1), (1, 8), (2, 5)])
def test_shared_groups(sa, kv, D, Hkv, rep):
    prompts = [200, 64, 30, 129, 640]
    tails = [[1, 5, 70], [0, 3], [4, 4], [9], [0, 0, 1, 40, 64, 65, 3, 2, 90]]
    r, groups = shared_rows(sa, kv, Hkv, D, prompts, tails, 6)
    n = sum(groups)
    q = r.query(n, rep)
    want = r.want(q, range(n), D ** -0.5)
    close(r.cache.decode_shared(0, q, D ** -0.5, groups), want)
    close(r.cache.decode_shared(0, q, D ** -0.5), want)                   # one group: nothing in common
    close(r.cache.decode_shared(0, q, D ** -0.5, [1] * n), want)          # no group
    ids = list(range(n))[::-1]
    close(r.cache.decode_shared(0, q, D ** -0.5, groups[::-1], seq_ids=ids), r.want(q, ids, D ** -0.5))
    for row in range(n):
        r.cache.reserve(row, r.cache.length(row) + 1)
        r.append(row, 1, commit=False)
    close(r.cache.decode_shared(0, q, D ** -0.5, groups, n_pending=1), r.want(q, range(n), D ** -0.5))
    r.cache.close()


@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("rows,rep", [(8, 2), (16, 2), (17, 2), (32, 2), (33, 2), (64, 2), (64, 8), (70, 2), (130, 1)])
def test_shared_row_counts(sa, kv, rows, rep):
    """Every split of a workgroup's waves over query rows and keys, groups of
    several row blocks, and more rows than one launch takes."""
    D, Hkv = 128, 1
    r, groups = shared_rows(sa, kv, Hkv, D, [1000, 70], [[i % 40 for i in range(rows)], [3, 1]], 7)
    n = sum(groups)
    q = r.query(n, rep)
    want = r.want(q, range(n), D ** -0.5)
    for kv_block in (0, 64, 256):
        sa.set_attention_blocks(0, kv_block)
        try:
            close(r.cache.decode_shared(0, q, D ** -0.5, groups), want)
        finally:
            sa.set_attention_blocks(0, 0)
    r.cache.close()


def test_shared_equals_plain_decode(sa):
    """The same rows through the ordinary paged decode."""
    r, groups = shared_rows(sa, "bf16", 2, 128, [2000], [[7, 100, 3, 64]], 8)
    q = r.query(4, 2)
    got = r.cache.decode_shared(0, q, 0.09, groups)
    plain = r.cache.decode(0, q, 0.09)
    assert (got - plain).norm() <= 4e-6 * plain.norm()
    r.cache.close()


@pytest.mark.parametrize("form", ["window", "shared"])
def test_refusals(sa, form):
    r = Rows(sa, "f32", 2, 64, [100, 700], 9)
    lib, c = sa.lib(), r.cache
    q = r.query(2, 2)
    out = torch.full_like(q, 7.0)
    need = c.decode_window_ws_bytes(2, 4, 600, 4) if form == "window" else c.decode_shared_ws_bytes(2, 4)
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    ints = lambda *v: (C.c_int32 * len(v))(*v)  # noqa: E731

    def call(h=c.handle, layer=0, q=q.data_ptr(), n=2, ids=None, Hq=4, pend=0, window=600, sink=4, out=out.data_ptr(),
             ws=ws.data_ptr(), nb=need, sizes=None, ng=0):
        if form == "window":
            return lib.sa_paged_decode_window(h, layer, q, n, ids, Hq, pend, window, sink, 0.125, out, ws, nb, None)
        return lib.sa_paged_decode_shared(h, layer, q, n, ids, sizes, ng, Hq, pend, 0.125, out, ws, nb, None)

    assert call(h=None) == sa.SA_EINVAL
    assert call(layer=1) == sa.SA_ERANGE and call(layer=-1) == sa.SA_ERANGE
    assert call(q=None) == sa.SA_EINVAL and call(out=None) == sa.SA_EINVAL
    assert call(n=0) == sa.SA_EINVAL and call(n=-1) == sa.SA_EINVAL and call(n=3) == sa.SA_ERANGE
    assert call(ids=ints(0, 2)) == sa.SA_ERANGE and call(ids=ints(-1, 0)) == sa.SA_ERANGE
    assert call(Hq=3) == sa.SA_EINVAL and call(Hq=0) == sa.SA_EINVAL and call(Hq=130) == sa.SA_EINVAL
    assert call(pend=-1) == sa.SA_EINVAL and call(pend=2000) == sa.SA_ERANGE
    assert call(q=q.data_ptr() + 4) == sa.SA_EINVAL and call(out=out.data_ptr() + 8) == sa.SA_EINVAL
    assert call(ws=ws.data_ptr() + 4) == sa.SA_EINVAL
    assert call(nb=16) == sa.SA_ENOMEM and call(ws=None, nb=0) == sa.SA_ENOMEM
    if form == "window":
        assert call(window=0) == sa.SA_EINVAL and call(window=-3) == sa.SA_EINVAL and call(sink=-1) == sa.SA_EINVAL
    else:
        assert call(sizes=ints(1), ng=1) == sa.SA_EINVAL and call(sizes=ints(1, 2), ng=2) == sa.SA_EINVAL
        assert call(sizes=ints(2, 0), ng=2) == sa.SA_EINVAL and call(sizes=ints(3, -1), ng=2) == sa.SA_EINVAL
        assert call(sizes=None, ng=1) == sa.SA_EINVAL and call(sizes=ints(2), ng=0) == sa.SA_EINVAL
    torch.cuda.synchronize()
    assert (out == 7.0).all()      # a refused call enqueues nothing
    assert call() == sa.SA_OK
    torch.cuda.synchronize()
    small = sa.KVCache(1, 2, 32, 1, 1, 1)
    with pytest.raises(sa.SaError, match="head_dim"):
        small.decode_shared(0, torch.zeros(1, 2, 32, device="cuda"), 1.0)
    with pytest.raises(sa.SaError, match="head_dim"):
        small.decode_window(0, torch.zeros(1, 2, 32, device="cuda"), 1.0, 5)
    with pytest.raises(ValueError):
        c.decode_window(0, q, 1.0, 5, out=torch.empty(1, 4, 64, device="cuda"))
    with pytest.raises(ValueError):
        c.decode_shared(0, q.double(), 1.0)
    small.close()
    c.close()


def test_ws_bytes_of_bad_arguments(sa):
    assert sa.lib().sa_paged_decode_window_ws_bytes(None, 1, 1, 1, 0) == 0
    assert sa.lib().sa_paged_decode_shared_ws_bytes(None, 1, 1) == 0


@pytest.mark.parametrize("kv", ["f32", "bf16"])
def test_graph_replays(sa, kv):
    """Both forms captured on a stream of their own, each with its workspace,
    and replayed between eager calls on the current one."""
    r, groups = shared_rows(sa, kv, 2, 128, [900], [[7, 100, 3, 64]], 10)
    q = r.query(4, 2)
    c = r.cache
    outs = [torch.empty_like(q) for _ in range(2)]
    wss = [torch.empty(c.decode_shared_ws_bytes(4, 4), dtype=torch.uint8, device="cuda"),
           torch.empty(c.decode_window_ws_bytes(4, 4, 300, 4), dtype=torch.uint8, device="cuda")]

    def both():
        c.decode_shared(0, q, 0.09, groups, out=outs[0], ws=wss[0])
        c.decode_window(0, q, 0.09, 300, 4, out=outs[1], ws=wss[1])

    both()
    torch.cuda.synchronize()
    want = [o.clone() for o in outs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for _ in range(3):
        for o in outs:
            o.fill_(float("nan"))
        for w in wss:
            w.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
        assert torch.equal(c.decode_shared(0, q, 0.09, groups), want[0])
        assert torch.equal(c.decode_window(0, q, 0.09, 300, 4), want[1])
    del graph
    c.close()


def test_streams_at_once(sa):
    """Calls on two streams with workspaces of their own."""
    r = Rows(sa, "bf16", 2, 128, [3000, 100, 5000, 1], 11)
    q = r.query(4, 2)
    want = r.want(q, range(4), 0.1, 2000, 4)
    full = r.want(q, range(4), 0.1)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        with torch.cuda.stream(streams[0]):
            outs.append((r.cache.decode_window(0, q, 0.1, 2000, 4), want))
        with torch.cuda.stream(streams[1]):
            outs.append((r.cache.decode_shared(0, q, 0.1), full))
    torch.cuda.synchronize()
    for got, w in outs:
        close(got, w)
    r.cache.close()


def same_with_infinities(got, want):
    """Of one kind everywhere; finite values within 1e-4, or within 3e-4 of
    themselves where one value near fp32's limit makes them (twice the error of
    its weight, which a score's 5.6e-5 and a normaliser's make)."""
    got, want = got.double(), want.double()
    for kind in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(kind(got), kind(want)), (kind, kind(got).sum().item(), kind(want).sum().item())
        assert kind(want).any()
    fine = torch.isfinite(want)
    over = ((got - want).abs()[fine] / torch.clamp(3e-4 * want.abs()[fine], min=1e-4)).max().item()
    assert over <= 1, over


@pytest.mark.parametrize("kv", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows", [2, 8, 12, 20, 40, 64])
def test_infinities_in_sight(sa, kv, D, rows):
    """Infinite keys and values, and values near the types' limits, that the rows
    see: what the formula makes of them, whichever split of the waves a number of
    rows takes, and as the ordinary paged decode has it."""
    P, Hkv, rep = 300, 2, 2
    r = Rows(sa, kv, Hkv, D, [P] + [0] * (rows - 1), 20 + rows, spare=12 * rows, width=8)
    k, v = r.k[0], r.v[0]
    v[70, :, 3], v[71, :, 5] = np.inf, -np.inf
    v[299, :, 6], v[0, :, 7], v[40, :, 8] = np.inf, -np.inf, 3.4e38 if kv == "f32" else 3.3e38
    v[90, :, 10], v[91, :, 10] = np.inf, -np.inf        # NaN
    k[33, 0, 0] = np.inf                                # head 0: a weight of 0, or NaN, by the sign of q
    r.cache.set_len(0, 0)
    r.cache.append(0, None, k[None], v[None], seq_ids=[0])
    r.cache.commit(P, seqs=[0])
    r.k[0], r.v[0] = (x.to(r.dtype).float() for x in (k, v))      # as they are stored
    for i in range(1, rows):
        r.fork(i, 0, P)
    for i in range(rows):
        r.cache.reserve(i, P + 5)
        r.append(i, 1 + i % 5)
    q = r.query(rows, rep)
    ids = range(rows)
    scale = D ** -0.5
    for kv_block in (0, 64):
        sa.set_attention_blocks(0, kv_block)
        try:
            want = r.want(q, ids, scale)
            same_with_infinities(r.cache.decode_shared(0, q, scale), want)
            same_with_infinities(r.cache.decode_shared(0, q, scale, [1] * rows), want)
            same_with_infinities(r.cache.decode(0, q, scale), want)
            for window, sink in ((1000, 0), (260, 5), (6, 92)):
                same_with_infinities(r.cache.decode_window(0, q, scale, window, sink), r.want(q, ids, scale, window, sink))
        finally:
            sa.set_attention_blocks(0, 0)
    r.cache.close()
