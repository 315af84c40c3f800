"""GPU tests of causal prefill with a sliding window and sinks against the
masked softmax in 64 bits.

fp32: max-abs 1e-4 and relative L2 2e-6, the bound of the fp32 attention tests
(test_gpu_ranges.py derives it).  bf16: each weight is rounded by at most 2^-9
of itself and each output by 2^-9, so an output is off by at most 2^-9 of
sum_j p_j |v_j| / sum_j p_j, and by 2^-8 of that with the rounded sums, plus
half a step of itself; with fp32 scores that adds 1e-4.
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def reference(q, k, v, scale, window, sink):
    """(out, sum of weights x |v|) in 64 bits."""
    B, Hq, L, D = q.shape
    rep = Hq // k.shape[1]
    i, j = torch.arange(L, device=q.device)[:, None], torch.arange(L, device=q.device)[None]
    unseen = (j > i) | ((i - j >= window) & (j >= sink))
    out, mag = [], []
    for b in range(B):
        for h in range(Hq):
            s = q[b, h].double() @ k[b, h // rep].double().T * scale
            p = torch.softmax(s.masked_fill(unseen, float("-inf")), -1)
            out.append(p @ v[b, h // rep].double())
            mag.append(p @ v[b, h // rep].double().abs())
    return torch.stack(out).reshape(q.shape), torch.stack(mag).reshape(q.shape)


def compare(got, want, mag):
    assert torch.isfinite(got).all()
    err = (got.double() - want).abs()
    if got.dtype == torch.float32:
        assert err.max().item() <= 1e-4
        assert err.norm().item() <= 2e-6 * want.norm().item()
    else:
        assert (err <= 2.0 ** -8 * mag + 2.0 ** -9 * want.abs() + 1e-4).all(), (err - 2.0 ** -8 * mag).max().item()
        assert err.norm().item() <= 4e-3 * want.norm().item()


def tensors(dtype, B, Hq, Hkv, L, D, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(B, H, L, D, device="cuda", generator=gen).to(DT[dtype]) for H in (Hq, Hkv, Hkv)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("L", [1, 2, 15, 16, 31, 33, 63, 64, 65, 127, 129, 200, 257, 500])
def test_lengths(sa, dtype, D, L):
    q, k, v = tensors(dtype, 2, 4, 2, L, D, L)
    for window, sink in ((1, 0), (40, 3), (64, 64), (100, 0), (1000, 4)):
        got = sa.prefill_window(q, k, v, D ** -0.5, window, sink)
        compare(got, *reference(q, k, v, D ** -0.5, window, sink))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("window", [1, 31, 32, 33, 63, 64, 65, 128, 300, 699, 700, 2 ** 31 - 1])
@pytest.mark.parametrize("sink", [0, 1, 5, 32, 64, 65, 130, 650, 2 ** 31 - 1])
def test_edges(sa, dtype, window, sink):
    q, k, v = tensors(dtype, 1, 2, 1, 700, 64, 3)
    compare(sa.prefill_window(q, k, v, 0.125, window, sink), *reference(q, k, v, 0.125, window, sink))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,Hq,Hkv,L", [(1, 16, 8, 1500), (3, 8, 8, 300), (2, 6, 2, 300), (1, 32, 4, 900), (8, 8, 1, 100),
                                        (1, 16, 1, 400), (5, 5, 5, 130), (1, 12, 1, 333), (40, 16, 8, 200)])
def test_heads(sa, dtype, B, Hq, Hkv, L):
    """Grids with and without a map of KV heads to XCDs, four and eight waves,
    head groups that a workgroup serves whole or in parts."""
    q, k, v = tensors(dtype, B, Hq, Hkv, L, 128, 5)
    compare(sa.prefill_window(q, k, v, -0.09, 150, 4), *reference(q, k, v, -0.09, 150, 4))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_token_major_and_broadcast(sa, dtype):
    """[B, L, H, D] projections as views, batches that share K and V, and a
    padded output whose other places stay as they are."""
    B, L, Hq, Hkv, D = 3, 210, 4, 2, 64
    gen = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(B, L, Hq + 2 * Hkv, D, device="cuda", generator=gen).to(DT[dtype])
    q, k, v = (t.transpose(1, 2) for t in x.split([Hq, Hkv, Hkv], 2))
    buf = torch.full((B, L, Hq + 1, D + 64), 5.0, device="cuda", dtype=DT[dtype])
    out = buf[:, :, :Hq, :D].transpose(1, 2)
    got = sa.prefill_window(q, k, v, 0.1, 50, 2, out=out)
    compare(got, *reference(q, k, v, 0.1, 50, 2))
    assert (buf[:, :, Hq] == 5).all() and (buf[:, :, :, D:] == 5).all()
    k1, v1 = (t[:1].expand(B, -1, -1, -1) for t in (k, v))
    compare(sa.prefill_window(q, k1, v1, 0.1, 50, 2), *reference(q, k1, v1, 0.1, 50, 2))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_large_scores(sa, dtype):
    """Scores that grow along the prompt to hundreds: the running max is raised
    again and again; near one-hot weights pass a value through."""
    q, k, v = tensors(dtype, 1, 2, 1, 600, 128, 7)
    k = k * torch.linspace(0.1, 8, 600, device="cuda").to(k.dtype)[:, None]
    want, mag = reference(q, k, v, 1.0, 200, 4)
    got = sa.prefill_window(q, k, v, 1.0, 200, 4)
    assert torch.isfinite(got).all()
    # scores up to 128 x 8 x 3: rounded by 131 x 2^-24 x 3000 at most, a weight by 2.4e-2
    assert (got.double() - want).norm().item() <= 2.4e-2 * want.norm().item()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_whole_prompt_equals_causal(sa, dtype):
    q, k, v = tensors(dtype, 1, 16, 8, 777, 128, 8)
    got = sa.prefill_window(q, k, v, 0.088, 777)
    full = sa.prefill_causal(q, k, v, 0.088)
    assert (got.float() - full).norm() <= (2e-6 if dtype == "f32" else 5e-3) * full.norm()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_prompt_then_decode(sa, dtype):
    """A streaming session: the prompt's last row through prefill_window, the
    same token through decode_window over the cache that holds the prompt."""
    L, window, sink = 500, 120, 4
    q, k, v = tensors(dtype, 1, 4, 2, L, 64, 9)
    out = sa.prefill_window(q, k, v, 0.125, window, sink)
    cache = sa.KVCache(1, 2, 64, 1, 9, 9, sa.SA_DTYPE_F32 if dtype == "f32" else sa.SA_DTYPE_BF16)
    cache.reserve(0, L)
    cache.append(0, None, *(t.transpose(1, 2).float().contiguous() for t in (k, v)))
    cache.commit(L, n_seqs=1)
    last = cache.decode_window(0, q[:, :, -1].float().contiguous(), 0.125, window, sink)
    assert (last - out[:, :, -1].float()).norm() <= (4e-6 if dtype == "f32" else 5e-3) * last.norm()
    cache.close()


def test_refusals(sa):
    import ctypes as C
    lib = sa.lib()
    q, k, v = tensors("f32", 1, 4, 2, 100, 64, 10)
    out = torch.full_like(q, 7.0)
    st = lambda *x: C.cast((C.c_int64 * 3)(*x), C.c_void_p)  # noqa: E731

    def call(q=q.data_ptr(), k=k.data_ptr(), dt=0, B=1, Hq=4, Hkv=2, L=100, D=64, qs=None, ks=None, os=None, window=5,
             sink=1, out=out.data_ptr()):
        return lib.sa_prefill_window(q, k, v.data_ptr(), dt, B, Hq, Hkv, L, D, qs, ks, os, window, sink, 0.125, out, None)

    good = st(25600, 6400, 64)
    for bad in (dict(q=None), dict(out=None), dict(dt=2), dict(B=0), dict(Hq=3), dict(Hkv=0), dict(L=-1), dict(D=32),
                dict(D=96), dict(window=0), dict(window=-1), dict(sink=-1), dict(q=q.data_ptr() + 4), dict(qs=good),
                dict(qs=good, ks=good), dict(qs=good, ks=good, os=st(25600, 6400, 65)),
                dict(qs=st(-64, 6400, 64), ks=good, os=good), dict(L=(1 << 30) + 1), dict(k=k.data_ptr() + 8)):
        assert call(**bad) == sa.SA_EINVAL, bad
        assert lib.sa_last_error()
    torch.cuda.synchronize()
    assert (out == 7).all()
    assert call(L=0, q=None) == sa.SA_OK and call() == sa.SA_OK
    for bad in ((q, k, v[:, :, :50]), (q.double(), k, v), (q, k.bfloat16(), v), (q[..., ::2], k[..., ::2], v[..., ::2]),
                (q[0], k[0], v[0])):
        with pytest.raises(ValueError):
            sa.prefill_window(*bad, 1.0, 5)
    assert sa.prefill_window(q[:, :, :0], k[:, :, :0], v[:, :, :0], 1.0, 5).shape == (1, 4, 0, 64)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_graph_replays_and_streams(sa, dtype):
    q, k, v = tensors(dtype, 1, 16, 8, 400, 128, 11)
    want = sa.prefill_window(q, k, v, 0.09, 100, 4)
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        sa.prefill_window(q, k, v, 0.09, 100, 4, out=out)
    side = torch.cuda.Stream()
    for _ in range(3):
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        other = sa.prefill_window(q, k, v, 0.09, 100, 4, stream=side)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(other, want)
    del graph


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,Hq,Hkv,L,D,window,sink", [(1, 4, 2, 200, 64, 40, 3), (1, 4, 2, 200, 128, 40, 120),
                                                      (40, 16, 8, 200, 64, 1000, 0), (9, 16, 8, 460, 128, 150, 4)])
def test_not_finite(sa, dtype, B, Hq, Hkv, L, D, window, sink):
    """NaN and infinite keys and values, a padded tail among them: queries that do
    not see them are untouched, others get what the formula makes of them."""
    q, k, v = tensors(dtype, B, Hq, Hkv, L, D, 12)
    k[:, :, L - 30:], v[:, :, L - 30:] = float("nan"), float("nan")      # padding behind the prompts
    v[:, :, 20, 3], v[:, :, 70, 5] = float("inf"), -float("inf")
    v[:, :, 100, 7], v[:, :, 101, 7] = float("inf"), -float("inf")       # NaN for who sees both
    v[:, :, 130, 9] = float("nan")
    k[:, :, 110, 0] = float("inf")                                       # a weight of 0, or NaN, by the sign of q
    i, j = torch.arange(L, device="cuda")[:, None], torch.arange(L, device="cuda")[None]
    unseen = (j > i) | ((i - j >= window) & (j >= sink))
    before = [t.clone() for t in (q, k, v)]
    got = sa.prefill_window(q, k, v, 0.1, window, sink)
    for b, h in {(0, 0), (B - 1, Hq - 1), (B // 2, Hq // 2)}:
        s = (q[b, h].double() @ k[b, h * Hkv // Hq].double().T * 0.1).masked_fill(unseen, float("-inf"))
        p = torch.softmax(s, -1)
        vd = v[b, h * Hkv // Hq].double()
        want, mag = torch.empty(L, D, device="cuda", dtype=torch.float64), torch.empty(L, D, device="cuda", dtype=torch.float64)
        for r in range(L):
            see = ~unseen[r]
            want[r], mag[r] = p[r][see] @ vd[see], p[r][see] @ vd[see].abs()
        g = got[b, h].double()
        for kind in (torch.isnan, torch.isposinf, torch.isneginf):
            assert torch.equal(kind(g), kind(want)), (kind, (kind(g) != kind(want)).nonzero()[:4].tolist())
        fine = torch.isfinite(want)
        assert fine[:20].all() and not fine[L - 30:].any()
        bound = 1e-4 + (0.0 if dtype == "f32" else 2.0 ** -8 * mag + 2.0 ** -9 * want.abs())
        assert ((g - want).abs() <= bound)[fine].all()
    assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip((q, k, v), before))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
def test_not_finite_in_views(sa, dtype, D):
    """The same through token-major views, a negative scale and a padded output,
    whose other places stay as they are: every query sees an infinite value, so
    that all of its columns are computed anew."""
    B, L, Hq, Hkv, window, sink, scale = 3, 210, 4, 2, 50, 2, -0.1
    gen = torch.Generator(device="cuda").manual_seed(13)
    x = torch.randn(B, L, Hq + 2 * Hkv, D, device="cuda", generator=gen).to(DT[dtype])
    q, k, v = (t.transpose(1, 2) for t in x.split([Hq, Hkv, Hkv], 2))
    v[:, :, 0, 11] = float("inf")                      # a sink
    buf = torch.full((B, L, Hq + 1, D + 64), 5.0, device="cuda", dtype=DT[dtype])
    out = buf[:, :, :Hq, :D].transpose(1, 2)
    got = sa.prefill_window(q, k, v, scale, window, sink, out=out)
    assert torch.isposinf(got[..., 11]).all()
    rest = [c for c in range(D) if c != 11]
    clean = v.clone()
    clean[:, :, 0, 11] = 0
    want, mag = reference(q, k, clean, scale, window, sink)
    compare(got[..., rest], want[..., rest], mag[..., rest])
    assert (buf[:, :, Hq] == 5).all() and (buf[:, :, :, D:] == 5).all()
    k1, v1 = (t[:1].expand(B, -1, -1, -1) for t in (k, v))
    want, mag = reference(q, k1, clean[:1].expand(B, -1, -1, -1), scale, window, sink)
    got = sa.prefill_window(q, k1, v1, scale, window, sink)
    assert torch.isposinf(got[..., 11]).all()
    compare(got[..., rest], want[..., rest], mag[..., rest])
