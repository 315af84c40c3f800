"""GPU tests of how the windowed, shared-prefix and beam-search calls sit in a
program: outputs and workspaces made on the stream that the call runs on,
tensors of another device, sizes beyond a C int, refusals of a step."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def filled_cache(sa, rows, n):
    c = sa.KVCache(1, 2, 64, rows, (n + 64) // 64, rows * ((n + 64) // 64), sa.SA_DTYPE_BF16)
    gen = torch.Generator(device="cuda").manual_seed(n)
    for r in range(rows):
        c.reserve(r, n + 1)
    c.append(0, None, *(torch.randn(rows, n, 2, 64, device="cuda", generator=gen) for _ in range(2)))
    c.commit(n, n_seqs=rows)
    return c


def calls(sa):
    """Each operator as a call(stream) whose output takes 4 MiB, or a little."""
    c = filled_cache(sa, 1024, 5)
    q = torch.randn(1024, 16, 64, device="cuda")
    qw, kw = torch.randn(1, 16, 1024, 64, device="cuda"), torch.randn(1, 2, 1024, 64, device="cuda")
    x, s = torch.randn(2, 4, 1000, device="cuda"), torch.zeros(2, 4, device="cuda")
    return c, [(q.numel() * 4, lambda st: c.decode_window(0, q, 0.1, 3, 1, stream=st)),
               (q.numel() * 4, lambda st: c.decode_shared(0, q, 0.1, stream=st)),
               (q.numel() * 4, lambda st: sa.prefill_window(qw, kw, kw, 0.1, 100, 2, stream=st)),
               (2 * 8 * 4, lambda st: sa.beam_select(x, s, 8, stream=st))]


@pytest.mark.parametrize("raw", [False, True])
def test_outputs_belong_to_the_calls_stream(sa, raw):
    c, todo = calls(sa)
    side = torch.cuda.Stream()
    for nbytes, call in todo:
        want = call(None)
        torch.cuda.synchronize()
        # memory that the current stream has just given back, perhaps with work
        # still reading it, is not another stream's to write
        old = [torch.empty(nbytes, dtype=torch.uint8, device="cuda") for _ in range(8)]
        freed = {t.data_ptr() for t in old}
        del old
        got = call(side.cuda_stream if raw else side)
        side.synchronize()
        for g, w in zip(got if isinstance(got, tuple) else [got], want if isinstance(want, tuple) else [want]):
            assert g.data_ptr() not in freed
            assert torch.equal(g, w)
    c.close()


def test_other_devices(sa, monkeypatch):
    c, todo = calls(sa)
    q = torch.randn(1, 16, 64)
    for bad in (lambda: c.decode_window(0, q, 0.1, 3), lambda: c.decode_shared(0, q, 0.1),
                lambda: c.decode_shared(0, q.cuda(), 0.1, ws=torch.empty(1 << 20, dtype=torch.uint8)),
                lambda: sa.prefill_window(q[None], q[None], q[None], 0.1, 5),
                lambda: sa.prefill_window(q[None].cuda(), q[None].cuda(), q[None], 0.1, 5),
                lambda: sa.beam_select(torch.zeros(1, 1, 9), torch.zeros(1, 1), 2),
                lambda: sa.beam_select(torch.zeros(1, 1, 9).cuda(), torch.zeros(1, 1), 2)):
        with pytest.raises(ValueError):
            bad()
    # tensors on device 0 while another one is current
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    for _, call in todo:
        with pytest.raises(ValueError):
            call(None)
    monkeypatch.undo()
    c.close()


def test_sizes_beyond_a_c_int(sa):
    """A window without end, as Python writes it."""
    c = filled_cache(sa, 3, 200)
    q = torch.randn(3, 4, 64, device="cuda")
    full = c.decode_window(0, q, 0.1, 201)
    for window, sink in ((2**32 + 1, 0), (10**18, 2**40), (1, 2**33 + 1)):
        assert torch.equal(c.decode_window(0, q, 0.1, window, sink), full)
    with pytest.raises(RuntimeError):
        c.decode_window(0, q, 0.1, 0)
    qw, kw = torch.randn(1, 4, 300, 64, device="cuda"), torch.randn(1, 2, 300, 64, device="cuda")
    full = sa.prefill_window(qw, kw, kw, 0.1, 300)
    for window, sink in ((2**32 + 1, 0), (2**31, 2**32), (1, 2**33 + 1)):
        assert torch.equal(sa.prefill_window(qw, kw, kw, 0.1, window, sink), full)
    c.close()


def test_scores_in_place(sa):
    """A selection of as many as there are beams, into the scores themselves."""
    x = torch.randn(5, 6, 4001, device="cuda")
    s = -torch.rand(5, 6, device="cuda")
    want = sa.beam_select(x, s, 6)
    out = (s, *(torch.empty(5, 6, dtype=torch.int32, device="cuda") for _ in range(2)))
    got = sa.beam_select(x, s, 6, out=out)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("interleave", ["0", "1"])
def test_steps_into_shared_pages_are_refused_whole(sa, monkeypatch, interleave):
    """Rows whose next token would fall into a shared page: no other row of the
    step gets a token either, in a one-layer model whose halves overlap."""
    monkeypatch.setenv("SA_DECODE_INTERLEAVE", interleave)
    model = sa.Qwen3(4, 200, num_layers=1, hidden=256, intermediate=512, vocab=1024, n_q_heads=4, n_kv_heads=2,
                     head_dim=64, rms_eps=1e-6, rope_theta=1e6)
    model.init_random(3, 0.1)
    cache = sa.KVCache(1, 2, 64, 4, 3, 12, sa.SA_DTYPE_F32)
    for r in range(4):
        cache.reserve(r, 100)
    tokens = torch.zeros(4, 64, dtype=torch.int32, device="cuda")
    model.prefill(cache, tokens)
    cache.fork(3, 2, 64)
    cache.reserve(3, 100)
    cache.set_len(3, 60)
    one = torch.zeros(4, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="shares"):
        model.decode_step(cache, one)
    with pytest.raises(RuntimeError, match="shares"):
        model.beam_step(cache, one.view(1, 4), torch.zeros(1, 4, device="cuda"), 4)
    assert [cache.length(r) for r in range(4)] == [64, 64, 64, 60]
    for r in range(4):
        cache.set_len(r, 0)
    with pytest.raises(RuntimeError, match="shares"):
        model.prefill(cache, tokens)
    assert [cache.length(r) for r in range(4)] == [0] * 4
    cache.fork(3, 2, 0)             # pages of its own again
    cache.reserve(3, 100)
    model.prefill(cache, tokens)
    model.decode_step(cache, one)
    torch.cuda.synchronize()
    assert [cache.length(r) for r in range(4)] == [65] * 4
    cache.close()
    model.close()


def test_small_workspaces_refuse_many_rows_whole(sa):
    """70 rows take two launches; the first would fit the workspace."""
    lens = [64] * 64 + [4000] * 6
    c = sa.KVCache(1, 1, 64, 70, 63, 64 + 6 * 63, sa.SA_DTYPE_BF16)
    for r, n in enumerate(lens):
        c.reserve(r, n)
        c.set_len(r, n)
    q = torch.randn(70, 4, 64, device="cuda")
    out = torch.full_like(q, 7.0)
    ws = torch.empty(4096, dtype=torch.uint8, device="cuda")
    for call in (lambda: c.decode_window(0, q, 0.1, 4000, out=out, ws=ws), lambda: c.decode_shared(0, q, 0.1, out=out, ws=ws)):
        with pytest.raises(RuntimeError, match="workspace"):
            call()
        torch.cuda.synchronize()
        assert (out == 7).all()
    c.close()


@pytest.mark.parametrize("P", [200, 4100])
def test_beam_step_replayed(sa, P):
    """A step captured into a graph and replayed from the state of the call, row
    by row (200 tokens) and over shared pages (4100)."""
    model = sa.Qwen3(4, P + 10, num_layers=2, hidden=256, intermediate=512, vocab=1024, n_q_heads=4, n_kv_heads=2,
                     head_dim=64, rms_eps=1e-6, rope_theta=1e6)
    model.init_random(7, 0.1)
    cache = sa.KVCache(2, 2, 64, 4, P // 64 + 1, 4 * (P // 64 + 1), sa.SA_DTYPE_BF16)
    cache.reserve(0, P)
    for layer in range(2):
        cache.append(layer, None, *(torch.randn(1, P, 2, 64, device="cuda") for _ in range(2)), seq_ids=[0])
    cache.commit(P, seqs=[0])
    for r in range(1, 4):
        cache.fork(r, 0, P)
    for r in range(4):
        cache.reserve(r, P + 1)
    tokens = torch.tensor([[5, 6, 7, 8]], dtype=torch.int32, device="cuda")
    scores = torch.tensor([[-1.0, -2.0, -3.0, -4.0]], device="cuda")
    out = (torch.empty(1, 8, device="cuda"), *(torch.empty(1, 8, dtype=torch.int32, device="cuda") for _ in range(2)))

    def back():
        for r in range(4):
            cache.set_len(r, P)

    want = [t.clone() for t in model.beam_step(cache, tokens, scores, 8, out=out)]
    back()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        model.beam_step(cache, tokens, scores, 8, out=out)
    for _ in range(3):
        back()
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        back()
        again = model.beam_step(cache, tokens, scores, 8)
        assert all(torch.equal(a, b) for a, b in zip(again, want))
    del graph
    cache.close()
    model.close()


@pytest.mark.parametrize("B,n", [(3, 6), (6, 3), (4, 64)])
def test_one_search_in_place(sa, B, n):
    """One search may select more or fewer than it has beams over its scores;
    several may not, and are refused with nothing written."""
    x = torch.randn(3, B, 4001, device="cuda")
    buf = -torch.rand(3 * max(B, n), device="cuda")
    s = buf[:B].view(1, B)
    want = sa.beam_select(x[:1], s, n)
    ints = [torch.full((3, n), 7, dtype=torch.int32, device="cuda") for _ in range(2)]
    got = sa.beam_select(x[:1], s, n, out=(buf[:n].view(1, n), *(t[:1] for t in ints)))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    before = buf.clone()
    for t in ints:
        t.fill_(7)
    with pytest.raises(RuntimeError, match="out_scores"):
        sa.beam_select(x, buf[:3 * B].view(3, B), n, out=(buf[:3 * n].view(3, n), *ints))
    torch.cuda.synchronize()
    assert torch.equal(buf, before) and all((t == 7).all() for t in ints)
