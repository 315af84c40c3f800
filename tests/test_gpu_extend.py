"""GPU tests of the attention of chunks of new tokens over a paged cache, of the
ragged append before it and of lengths set for many rows, against 64-bit
attention over what the cache holds.

Tolerances.  fp32: a score is a sum of at most 128 products of exact operands split
into terms, off by at most 131 x 2^-24 sum |q_d k_d| scale = 5.6e-5 for N(0,1) inputs,
an output by 9e-5: max-abs 1e-4; errors of random sign stay below 4e-6 in relative
L2.  bf16: the output's rounding, 2^-8 of its magnitude, and weights rounded to
bf16, each off by at most 2^-8 as is their sum: 2^-7 of sum w |v|, beside the 1e-4 of
the scores.
"""
from __future__ import annotations

import ctypes as C
import math

import pytest
import torch

from kv_rows import KV, Rows, attend, code

pytestmark = pytest.mark.gpu

PAIRS = [("f32", "f32"), ("f32", "bf16"), ("f32", "fp8"), ("bf16", "bf16"), ("bf16", "fp8")]
TYPE = {"f32": torch.float32, "bf16": torch.bfloat16}


def check(got, want, mag, l2=4e-6):
    assert got.isfinite().all()
    err = (got.double() - want).abs()
    if got.dtype == torch.float32:
        assert err.max().item() <= 1e-4, err.max().item()
        assert (err.norm() / want.norm()).item() <= l2, (err.norm() / want.norm()).item()
    else:
        over = (err - (2.0 ** -8 * want.abs() + 2.0 ** -7 * mag + 1e-4)).max().item()
        assert over <= 0, over
        assert (err.norm() / want.norm()).item() <= 2.0 ** -8


def check_all(rows, got, q, counts, lens, scale, ids=None):
    at = 0
    for i, n in enumerate(counts):
        if n:
            r = i if ids is None else ids[i]
            check(got[at:at + n], *attend(q[at:at + n], rows.k[r], rows.v[r], scale, lens[r]))
        at += n


SHAPES = [(16, 8, 128), (4, 4, 64), (8, 1, 128), (64, 1, 64), (6, 2, 64), (10, 2, 128)]


@pytest.mark.parametrize("q,kv", PAIRS)
@pytest.mark.parametrize("Hq,Hkv,D", SHAPES)
def test_ragged(sa, q, kv, Hq, Hkv, D):
    lens = [0, 0, 63, 64, 65, 130, 1000, 777, 5]
    counts = [1, 70, 1, 5, 64, 0, 3, 129, 2]
    rows = Rows(sa, kv, Hkv, D, lens, seed=Hq + D, room=130)
    rows.append(counts)
    x = rows.normal(sum(counts), Hq, D, dtype=TYPE[q])
    scale = 1 / math.sqrt(D)
    got = rows.cache.extend(0, x, scale, counts)
    check_all(rows, got, x, counts, lens, scale)


@pytest.mark.parametrize("q,kv", PAIRS)
@pytest.mark.parametrize("n,past", [(1, 0), (1, 4000), (5, 6001), (17, 2047), (256, 0), (300, 1500), (513, 63)])
def test_one_sequence(sa, q, kv, n, past):
    rows = Rows(sa, kv, 2, 128, [past], seed=n + past, room=n)
    rows.append([n])
    x = rows.normal(1, n, 4, 128, dtype=TYPE[q])
    got = rows.cache.extend(0, x, 0.088)
    check(got[0], *attend(x[0], rows.k[0], rows.v[0], 0.088, past))


@pytest.mark.parametrize("q,kv", PAIRS)
def test_many_sequences(sa, q, kv):
    """More than one launch takes, rows listed out of order and twice."""
    lens = [(i * 53) % 300 for i in range(70)]
    rows = Rows(sa, kv, 1, 64, lens, seed=11, room=4)
    rows.append([4] * 70)
    ids = list(range(69, -1, -1)) + [3, 3]
    counts = [i % 5 for i in range(72)]
    x = rows.normal(sum(counts), 2, 64, dtype=TYPE[q])
    got = rows.cache.extend(0, x, -0.2, counts, seq_ids=ids)
    check_all(rows, got, x, counts, lens, -0.2, ids)


@pytest.mark.parametrize("kv", KV)
def test_one_token_is_a_decode(sa, kv):
    lens = [1, 100, 64, 3000]
    rows = Rows(sa, kv, 2, 128, lens, seed=12, room=1)
    rows.append([1] * 4)
    x = rows.normal(4, 8, 128)
    got = rows.cache.extend(0, x, 0.1, [1] * 4)
    want = rows.cache.decode(0, x, 0.1, n_pending=1)
    assert (got - want).abs().max().item() <= 1e-5


@pytest.mark.parametrize("q,kv", PAIRS)
def test_a_prompt_in_chunks(sa, q, kv):
    """Chunks of a prompt, each over what is committed by then, give the rows of the whole prompt."""
    n, parts = 700, [1, 64, 300, 335]
    whole, pieces = (Rows(sa, kv, 2, 64, [0], seed=13, room=n) for _ in range(2))
    whole.append([n])
    x = whole.normal(n, 4, 64, dtype=TYPE[q])
    pieces.gen = torch.Generator(device="cuda").manual_seed(13)
    want = whole.cache.extend(0, x, 0.125, [n])
    k, v = (t.transpose(0, 1).contiguous() for t in _pending(whole, n))
    at = 0
    for c in parts:
        pieces.cache.append(0, None, k[at:at + c].contiguous(), v[at:at + c].contiguous(), counts=[c])
        got = pieces.cache.extend(0, x[at:at + c].contiguous(), 0.125, [c])
        tol = 2e-4 if q == "f32" else 2.0 ** -6 * 4
        assert (got.float() - want[at:at + c].float()).abs().max().item() <= tol
        pieces.cache.commit(c, n_seqs=1)
        at += c


def _pending(rows, n):
    rows.cache.commit(n, n_seqs=1)
    kv = rows.cache.gather(0, 0, n)
    rows.cache.set_len(0, 0)
    return kv


@pytest.mark.parametrize("q,kv", PAIRS)
@pytest.mark.parametrize("n,past", [(9, 200), (200, 90)])
def test_what_is_hidden_does_not_reach(sa, q, kv, n, past):
    """NaN and infinities in later tokens, appended or not, in places behind the chunk, and in sight of the last ones."""
    bad = n // 2
    rows = Rows(sa, kv, 2, 128, [past], seed=14, room=n + 20)

    def change(k, v):
        k[bad, 0], v[bad, 0] = float("nan"), float("inf")
        k[bad + 1, 1, 5], v[bad + 1, 1, 6] = float("inf"), float("nan")
    rows.append([n + 20], change=change)      # 20 more than the chunk
    x = rows.normal(n, 4, 128, dtype=TYPE[q])
    got = rows.cache.extend(0, x, 0.088, [n])
    check(got[:bad], *attend(x[:bad], rows.k[0], rows.v[0], 0.088, past))
    assert got[bad:, :2].isnan().all()                     # head 0's key is NaN from there on
    assert got[bad, 2:].isfinite().all()
    assert got[bad + 1:, 2:, 6].isnan().all()


def test_infinite_values_in_sight(sa):
    """fp32: an infinity that a token sees comes out, and a score of -inf hides its key."""
    rows = Rows(sa, "f32", 1, 64, [70], seed=15, room=10)

    def change(k, v):
        v[2, 0, 7] = float("inf")
        v[4, 0, 9] = -float("inf")
    rows.append([10], change=change)
    x = rows.normal(10, 2, 64)
    got = rows.cache.extend(0, x, 0.125, [10])
    assert got[:2].isfinite().all()
    assert (got[2:, :, 7] == float("inf")).all() and (got[4:, :, 9] == -float("inf")).all()
    fine = [d for d in range(64) if d not in (7, 9)]
    want = attend(x, rows.k[0], rows.v[0], 0.125, 70)[0]
    assert (got[..., fine].double() - want[..., fine]).abs().max().item() <= 1e-4


@pytest.mark.parametrize("q,kv", PAIRS)
@pytest.mark.parametrize("n", [6, 260])
def test_output_rows_behind_the_last_are_left(sa, q, kv, n):
    rows = Rows(sa, kv, 2, 64, [100, 10], seed=16, room=n)
    rows.append([n, n - 1])
    T = 2 * n - 1
    x = rows.normal(T, 4, 64, dtype=TYPE[q])
    buf = torch.full((T + 3, 4, 64), 7.0, dtype=TYPE[q], device="cuda")
    got = rows.cache.extend(0, x, 0.125, [n, n - 1], out=buf[:T])
    assert got.data_ptr() == buf.data_ptr() and (buf[T:] == 7).all()
    check_all(rows, got, x, [n, n - 1], [100, 10], 0.125)


@pytest.mark.parametrize("q,kv", PAIRS)
@pytest.mark.parametrize("n", [5, 300])
def test_captured_and_on_another_stream(sa, q, kv, n):
    rows = Rows(sa, kv, 2, 128, [900, 64], seed=17, room=n)
    rows.append([n, n])
    x = rows.normal(2 * n, 4, 128, dtype=TYPE[q])
    want = rows.cache.extend(0, x, 0.088, [n, n]).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = rows.cache.extend(0, x, 0.088, [n, n], stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    out = torch.empty_like(x)
    ws = torch.empty(max(16, rows.cache.extend_ws_bytes([n, n], 4)), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows.cache.extend(0, x, 0.088, [n, n], out=out, ws=ws)
    for _ in range(3):
        out.zero_()
        ws.fill_(255)                         # nothing is kept between calls
        rows.cache.extend(0, x, 0.088, [n, n])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_equal_calls_give_equal_bits(sa):
    rows = Rows(sa, "bf16", 8, 128, [3000, 100], seed=18, room=600)
    rows.append([600, 3])
    for dt in (torch.float32, torch.bfloat16):
        x = rows.normal(603, 16, 128, dtype=dt)
        first = rows.cache.extend(0, x, 0.088, [600, 3])
        assert all(torch.equal(rows.cache.extend(0, x, 0.088, [600, 3]), first) for _ in range(3))


@pytest.mark.parametrize("kv", KV)
def test_ragged_append_equals_one_by_one(sa, kv):
    """The same bits as a call per sequence, queries included."""
    D, Hq, Hkv, lens, counts = 64, 4, 2, [5, 0, 64, 100], [3, 0, 130, 1]
    a, b = (Rows(sa, kv, Hkv, D, lens, seed=19, room=130) for _ in range(2))
    T = sum(counts)
    q, k, v = a.normal(T, Hq, D), a.normal(T, Hkv, D), a.normal(T, Hkv, D)
    w = [1 + 0.1 * a.normal(D) for _ in range(2)]
    rope = sa.rope_tables(256, D)
    got = a.cache.append(0, q, k, v, *w, rope=rope, counts=counts)
    at = 0
    for r, n in enumerate(counts):
        if n:
            part = slice(at, at + n)
            one = b.cache.append(0, q[part][None].contiguous(), k[part][None].contiguous(), v[part][None].contiguous(),
                                 *w, rope=rope, seq_ids=[r])
            assert torch.equal(one[0], got[part])
            for c in (a.cache, b.cache):
                c.commit(n, seqs=[r])
            for x, y in zip(a.cache.gather(0, r, lens[r] + n), b.cache.gather(0, r, lens[r] + n)):
                assert torch.equal(x, y)
        at += n


def test_set_lens(sa):
    cache = sa.KVCache(1, 1, 64, 130, 2, 260)
    for r in range(130):
        cache.reserve(r, 128)
    ids = list(range(129, -1, -1))
    cache.set_lens(ids, [r % 129 for r in ids])
    lens = torch.as_tensor(sa._CudaArray(sa.lib().sa_kvcache_seq_lens(cache.handle), 130, "<i4"), device="cuda")
    assert lens.tolist() == [r % 129 for r in range(130)] == [cache.length(r) for r in range(130)]
    for ids, new in (([0, 0], [1, 1]), ([0, 200], [1, 1]), ([0, 1], [1, 129]), ([0, 1], [1, -1])):
        with pytest.raises(sa.SaError):
            cache.set_lens(ids, new)
    assert cache.length(0) == 0 and cache.length(1) == 1
    cache.set_lens([], [])
    with pytest.raises(ValueError):
        cache.set_lens([0], [])


def test_refusals(sa):
    rows = Rows(sa, "f32", 2, 64, [10, 20], seed=20, room=10)
    ext = rows.cache.extend
    x = rows.normal(6, 4, 64)
    with pytest.raises(sa.SaError, match="exceeds"):
        ext(0, rows.normal(60, 4, 64), 1.0, [60, 0])
    with pytest.raises(sa.SaError, match="bf16 queries"):
        ext(0, x.bfloat16(), 1.0, [3, 3])
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        ext(0, x.half(), 1.0, [3, 3])
    with pytest.raises(ValueError):
        ext(0, x, 1.0, [3, 2])
    with pytest.raises(ValueError):
        ext(0, x, 1.0)
    with pytest.raises(sa.SaError, match="counts"):
        ext(0, x, 1.0, [7, -1])
    with pytest.raises(sa.SaError, match="layer|Layer"):
        ext(1, x, 1.0, [3, 3])
    with pytest.raises(sa.SaError, match="head counts"):
        ext(0, rows.normal(6, 3, 64), 1.0, [3, 3])
    with pytest.raises(sa.SaError, match="out of range"):
        ext(0, x, 1.0, [3, 3], seq_ids=[0, 2])
    with pytest.raises(ValueError):
        ext(0, x[:, :, :32].contiguous(), 1.0, [3, 3])
    with pytest.raises(ValueError):
        ext(0, x, 1.0, [3, 3], out=torch.empty(6, 4, 64, device="cuda", dtype=torch.bfloat16))
    narrow = sa.KVCache(1, 1, 32, 1, 1, 1)
    narrow.reserve(0, 64)
    with pytest.raises(sa.SaError, match="head_dim"):
        narrow.extend(0, torch.zeros(1, 1, 32, device="cuda"), 1.0, [1])
    lib = sa.lib()
    one = (C.c_int32 * 2)(3, 3)
    args = lambda **k: [rows.cache.handle, 0, k.get("q", x.data_ptr()), k.get("dt", 0), k.get("n", 2), None,  # noqa: E731
                        k.get("counts", C.cast(one, C.c_void_p)), 4, 1.0, k.get("out", x.data_ptr()), None, 0, None]
    assert lib.sa_paged_extend(*args(q=x.data_ptr() + 4)) == sa.SA_EINVAL
    assert lib.sa_paged_extend(*args(q=None)) == sa.SA_EINVAL
    assert lib.sa_paged_extend(*args(dt=sa.SA_DTYPE_FP8)) == sa.SA_EINVAL
    assert lib.sa_paged_extend(*args(n=0)) == sa.SA_EINVAL
    assert lib.sa_paged_extend(*args(counts=None)) == sa.SA_EINVAL
    assert lib.sa_paged_extend(None, *args()[1:]) == sa.SA_EINVAL
    # a long context takes a workspace
    big = Rows(sa, "bf16", 1, 64, [4000], seed=21, room=10)
    big.append([10])
    y = big.normal(10, 1, 64)
    with pytest.raises(sa.SaError, match="workspace"):
        big.cache.extend(0, y, 1.0, [10], ws=torch.empty(16, dtype=torch.uint8, device="cuda"))
    ragged = dict(counts=[2, -1])
    with pytest.raises((sa.SaError, ValueError)):
        rows.cache.append(0, None, rows.normal(1, 2, 64), rows.normal(1, 2, 64), **ragged)
    with pytest.raises(sa.SaError, match="full"):
        rows.cache.append(0, None, rows.normal(100, 2, 64), rows.normal(100, 2, 64), counts=[100, 0])
    with pytest.raises(ValueError):
        rows.cache.append(0, None, rows.normal(5, 2, 64), rows.normal(5, 2, 64), counts=[2, 2])


def test_no_tokens_is_nothing_to_do(sa):
    rows = Rows(sa, "f32", 1, 64, [10, 0], seed=22)
    x = torch.empty(0, 2, 64, device="cuda")
    assert rows.cache.extend(0, x, 1.0, [0, 0]).shape == x.shape
    rows.cache.append(0, x, x[:, :1].contiguous(), x[:, :1].contiguous(), counts=[0, 0])
    assert rows.cache.length(0) == 10
    assert code(sa, "fp8") == sa.SA_DTYPE_FP8


def test_short_rows_of_many_sequences_take_no_workspace(sa):
    """Pages of one tile's tokens hold no more than one partial per row."""
    rows = Rows(sa, "bf16", 1, 64, [5] * 66, seed=23, room=2)
    rows.append([2] * 66)
    x = rows.normal(132, 1, 64)
    got = rows.cache.extend(0, x, 0.125, [2] * 66)
    check_all(rows, got, x, [2] * 66, [5] * 66, 0.125)


@pytest.mark.parametrize("q,kv", PAIRS)
def test_long_and_short_chunks_of_many_sequences(sa, q, kv):
    """Long chunks are taken together, out of rows that would otherwise be several launches'."""
    lens, counts = [64] * 256, [64, 1, 1, 1] * 64
    rows = Rows(sa, kv, 1, 64, lens, seed=24, room=64)
    rows.append(counts)
    x = rows.normal(sum(counts), 1, 64, dtype=TYPE[q])
    ws = torch.full((max(16, rows.cache.extend_ws_bytes(counts, 1)),), 255, dtype=torch.uint8, device="cuda")
    got = rows.cache.extend(0, x, 0.125, counts, ws=ws)
    check_all(rows, got, x, counts, lens, 0.125)


@pytest.mark.parametrize("q,kv", PAIRS)
@pytest.mark.parametrize("Hq,Hkv,D", [(3, 1, 64), (10, 2, 128), (12, 2, 64)])
@pytest.mark.parametrize("n,past", [(150, 100), (700, 37)])
def test_negative_scale_and_odd_groups(sa, q, kv, Hq, Hkv, D, n, past):
    rows = Rows(sa, kv, Hkv, D, [past], seed=25, room=n)
    rows.append([n])
    x = rows.normal(n, Hq, D, dtype=TYPE[q])
    got = rows.cache.extend(0, x, -0.11, [n])
    check(got, *attend(x, rows.k[0], rows.v[0], -0.11, past))


@pytest.mark.parametrize("q,kv", PAIRS)
def test_pages_beyond_32_bits(sa, q, kv):
    """Pools of more than 2^32 bytes: every row's pages lie anywhere in them."""
    spare = (1 << 32) // (64 * 8 * 128 * {"f32": 4, "bf16": 2, "fp8": 1}[kv]) + 4000
    rows = Rows(sa, kv, 8, 128, [5000, 700, 90], seed=26, room=300, spare=spare)
    counts = [5, 300, 2]
    rows.append(counts)
    x = rows.normal(sum(counts), 8, 128, dtype=TYPE[q])
    check_all(rows, rows.cache.extend(0, x, 0.088, counts), x, counts, [5000, 700, 90], 0.088)
    few = x[:1].float().repeat(3, 1, 1)
    got = rows.cache.decode(0, few, 0.088)
    for r, n in enumerate([5000, 700, 90]):
        check(got[r:r + 1], *attend(few[:1], rows.k[r][:n], rows.v[r][:n], 0.088, n - 1))
    k, v = rows.cache.gather(0, 0, 5000)
    assert torch.equal(k.transpose(0, 1).double(), rows.k[0][:5000]) and torch.equal(v.transpose(0, 1).double(), rows.v[0][:5000])


@pytest.mark.parametrize("q,kv", PAIRS)
def test_a_long_prompt_at_once(sa, q, kv):
    n = 70001
    rows = Rows(sa, kv, 1, 64, [0], seed=27, room=n)
    rows.append([n])
    x = rows.normal(n, 1, 64, dtype=TYPE[q])
    got = rows.cache.extend(0, x, 0.125, [n])
    for at in (0, 1, 63, 64, 127, 128, 255, 256, 30000, 65535, 65536, n - 2, n - 1):
        # A row's output accumulates 6 products for every 32 keys, each sum rounded by up
        # to half a step, 2^-24 of it, evenly distributed: sqrt(6 keys / 32 / 3) 2^-24 in
        # relative L2 (3.9e-6 at 70001 keys) beside the scores' 4e-6.
        l2 = 4e-6 + math.sqrt(6 * (at + 1) / 32 / 3) * 2.0 ** -24
        check(got[at:at + 1], *attend(x[at:at + 1], rows.k[0], rows.v[0], 0.125, at), l2)


@pytest.mark.parametrize("q,kv", PAIRS)
def test_two_graphs_on_one_workspace(sa, q, kv):
    rows = Rows(sa, kv, 2, 64, [2000, 300], seed=28, room=200)
    calls = [[200, 7], [3, 100]]
    rows.append([200, 100])
    need = max(rows.cache.extend_ws_bytes(c, 8) for c in calls)
    ws = torch.empty(max(16, need), dtype=torch.uint8, device="cuda")
    x = [rows.normal(sum(c), 8, 64, dtype=TYPE[q]) for c in calls]
    want = [rows.cache.extend(0, x[i], 0.125, c).clone() for i, c in enumerate(calls)]
    out, graphs = [torch.empty_like(t) for t in x], []
    for i, c in enumerate(calls):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            rows.cache.extend(0, x[i], 0.125, c, out=out[i], ws=ws)
    for _ in range(3):
        for i in (0, 1):
            out[i].zero_()
            graphs[i].replay()
            rows.cache.extend(0, x[1 - i], 0.125, calls[1 - i], ws=ws)
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(out, want))


@pytest.mark.parametrize("q,kv", PAIRS)
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 64), (16, 8, 128), (3, 1, 64)])
def test_chunks_of_unequal_lengths(sa, q, kv, Hq, Hkv, D):
    """Blocks in parts of all lengths, of sequences in no order of their lengths."""
    lens, counts = [3000, 40, 1500, 0, 700, 5000], [400, 300, 1, 200, 90, 33]
    rows = Rows(sa, kv, Hkv, D, lens, seed=29, room=400)
    rows.append(counts)
    x = rows.normal(sum(counts), Hq, D, dtype=TYPE[q])
    check_all(rows, rows.cache.extend(0, x, 0.1, counts), x, counts, lens, 0.1)


@pytest.mark.parametrize("q,kv", PAIRS)
def test_many_blocks_of_two_sequences(sa, q, kv):
    """More blocks than are put in order, and as many but one part each."""
    for n, past in ((5000, 100), (600, 0)):
        rows = Rows(sa, kv, 1, 64, [past, 0], seed=30, room=n)
        rows.append([n, n])
        x = rows.normal(2 * n, 8, 64, dtype=TYPE[q])
        got = rows.cache.extend(0, x, 0.125, [n, n])
        for r, first in ((0, 0), (1, n)):
            for at in (0, 1, 31, 32, 255, n // 2, n - 2, n - 1):
                i = first + at
                check(got[i:i + 1], *attend(x[i:i + 1], rows.k[r], rows.v[r], 0.125, (past, 0)[r] + at))
