"""GPU tests of caches in 8 bits: what an append stores (codes and scales), what
reading back gives, and every attention over such a cache against 64-bit
attention over what is held.

What is stored is compared bit for bit with the definition, computed in 64
bits.  Held values are exact in bf16, one term of the products, so outputs have the
bounds of the other fp32 attention tests: a score is a sum of 128 products off by
at most 131 x 2^-24 sum |q_d k_d| scale = 5.6e-5 for N(0,1) inputs, an output by 9e-5;
max-abs 1e-4, and 2e-6 relative L2 for errors of random sign.
"""
from __future__ import annotations

import math

import pytest
import torch

from kv_rows import Rows, attend, held_fp8, poison

pytestmark = pytest.mark.gpu


def check(got, want, tol=1e-4, l2=2e-6):
    assert got.isfinite().all()
    err = (got.double() - want).abs().max().item()
    rel = ((got.double() - want).norm() / want.norm()).item()
    assert err <= tol and rel <= l2, (err, rel)


def special_rows(D, n):
    """n rows: ordinary ones, and those where the format ends."""
    g = torch.Generator(device="cuda").manual_seed(D + n)
    x = torch.randn(n, D, device="cuda", generator=g)
    x *= torch.exp2(torch.randint(-30, 30, (n, 1), device="cuda", generator=g).float())
    t = torch.arange(D, device="cuda").float()
    rows = [torch.zeros(D), t.cpu() * 0 - 0.0, t.cpu() + 1, (t.cpu() - 60) * 3.5]
    top = [448.0, 448.0 * (1 + 2 ** -23), 447.99997, 2.0 ** -92 * 448, 448 * 2.0 ** -100, 448 * 2.0 ** -101, 3e-39, 1e-45,
           3.4028234663852886e38, 1.9375 * 2.0 ** 127, 1.75 * 2.0 ** 127, 1.0, 1.75, 1.7500001, 17.0, 2.0 ** -93]
    for m in top:
        r = torch.linspace(-1, 1, D, dtype=torch.float64) * m
        r[1] = m                      # the largest magnitude, and halves of steps below it
        r[2], r[3] = m * 17 / 448 * 4, m * 19 / 448 * 4
        rows.append(r.float())
    for bad in (float("nan"), float("inf"), -float("inf")):
        r = torch.linspace(-3, 3, D)
        r[5] = bad
        rows.append(r)
    rows.append(torch.full((D,), float("inf")))
    rows = torch.stack([r.float() for r in rows]).cuda()
    x[:len(rows)] = rows[:n]
    return x


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hkv,S,aligned", [(1, 40, True), (2, 300, True), (4, 700, True), (4, 700, False)])
def test_append_holds_the_definition(sa, D, Hkv, S, aligned):
    """Few head rows (a row per wave), many (16 bytes per lane), and pointers of any alignment."""
    cache = sa.KVCache(1, Hkv, D, 1, (S + 63) // 64, (S + 63) // 64, sa.SA_DTYPE_FP8)
    poison(sa, cache)
    cache.reserve(0, S)
    raw = [torch.empty(S * Hkv * D + 4, device="cuda") for _ in range(2)]
    k, v = (r[0 if aligned else 1:][:S * Hkv * D].view(1, S, Hkv, D) for r in raw)
    k.copy_(special_rows(D, S * Hkv).view(1, S, Hkv, D))
    v.copy_(k.flip(1) * 0.75)
    cache.append(0, None, k, v)
    cache.commit(S, n_seqs=1)
    for got, x, scales in zip(cache.gather(0, 0, S), (k, v), sa.kv_scale_views(cache, 0)):
        want, e = held_fp8(x[0].transpose(0, 1))
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.double().nan_to_num(0.0), want.nan_to_num(0.0))
        table = torch.tensor([[t // 64, t % 64] for t in range(S)], device="cuda")
        at = scales.view(-1, Hkv, 64)[table[:, 0], :, table[:, 1]]                 # [S, Hkv]
        assert torch.equal(at.long() - 127, e[..., 0].transpose(0, 1))
    # what is held is held again as it is
    again = sa.KVCache(1, Hkv, D, 1, (S + 63) // 64, (S + 63) // 64, sa.SA_DTYPE_FP8)
    again.reserve(0, S)
    kv = [x.transpose(0, 1).contiguous()[None] for x in cache.gather(0, 0, S)]
    again.append(0, None, *kv)
    again.commit(S, n_seqs=1)
    for a, b in zip(again.gather(0, 0, S), cache.gather(0, 0, S)):
        assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


def test_append_with_norm_and_rope_holds_what_they_give(sa):
    """The codes are those of the row that an fp32 cache gets."""
    D, Hkv, Hq, S = 128, 2, 4, 70
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(2, S, h, D, device="cuda", generator=g) for h in (Hq, Hkv, Hkv))
    w = [1 + 0.1 * torch.randn(D, device="cuda", generator=g) for _ in range(2)]
    rope = sa.rope_tables(256, D)
    got = []
    for dt in (sa.SA_DTYPE_F32, sa.SA_DTYPE_FP8):
        cache = sa.KVCache(1, Hkv, D, 2, 3, 6, dt)
        for r in range(2):
            cache.reserve(r, S + 5)
            cache.set_len(r, 5)
        qo = cache.append(0, q, k, v, *w, rope=rope)
        cache.commit(S, n_seqs=2)
        got.append((qo, [[x[:, 5:] for x in cache.gather(0, r, S + 5)] for r in range(2)]))
    assert torch.equal(got[0][0], got[1][0])
    for a, b in zip(got[0][1], got[1][1]):
        for x, y in zip(a, b):
            assert torch.equal(held_fp8(x)[0], y.double())


LENS = [1, 63, 64, 65, 700, 0, 2049, 5000]


@pytest.mark.parametrize("Hq,Hkv,D", [(16, 8, 128), (8, 8, 64), (12, 2, 128), (64, 1, 64), (32, 4, 64)])
def test_decode(sa, Hq, Hkv, D):
    rows = Rows(sa, "fp8", Hkv, D, LENS, seed=3)
    q = rows.normal(len(LENS), Hq, D)
    scale = 1 / math.sqrt(D)
    got = rows.cache.decode(0, q, scale)
    zero = LENS.index(0)
    assert (got[zero] == 0).all()
    for r, n in enumerate(LENS):
        if n:
            check(got[r], attend(q[r:r + 1], rows.k[r], rows.v[r], scale, n - 1)[0][0], l2=4e-6)


def test_decode_of_listed_rows_and_pending_tokens(sa):
    rows = Rows(sa, "fp8", 2, 128, [100, 300, 64], seed=4, room=3)
    rows.append([3, 3, 3])
    ids = [2, 0, 1, 2]
    q = rows.normal(4, 4, 128)
    got = rows.cache.decode(0, q, 0.1, n_pending=3, seq_ids=ids)
    for i, r in enumerate(ids):
        check(got[i], attend(q[i:i + 1], rows.k[r], rows.v[r], 0.1, len(rows.k[r]) - 1)[0][0])


def test_decode_of_more_rows_than_a_launch(sa):
    lens = [(37 * i) % 200 + 1 for i in range(70)]
    rows = Rows(sa, "fp8", 1, 64, lens, seed=5)
    q = rows.normal(70, 2, 64)
    got = rows.cache.decode(0, q, 0.125)
    for r in range(70):
        check(got[r], attend(q[r:r + 1], rows.k[r], rows.v[r], 0.125, lens[r] - 1)[0][0], l2=4e-6)


def test_window_and_shared_decode(sa):
    rows = Rows(sa, "fp8", 2, 128, [1000, 130, 64], seed=6)
    q = rows.normal(3, 4, 128)
    got = rows.cache.decode_window(0, q, 0.1, 200, 5)
    for r, n in enumerate([1000, 130, 64]):
        t = [i for i in range(n) if n - 1 - i < 200 or i < 5]
        check(got[r], attend(q[r:r + 1], rows.k[r][t], rows.v[r][t], 0.1, len(t) - 1)[0][0])
    fork = sa.KVCache(1, 2, 128, 3, 10, 40, sa.SA_DTYPE_FP8)
    poison(sa, fork)
    fork.reserve(0, 400)
    k, v = rows.normal(1, 300, 2, 128), rows.normal(1, 300, 2, 128)
    fork.append(0, None, k, v, seq_ids=[0])
    fork.commit(300, seqs=[0])
    fork.fork(1, 0, 300)
    fork.fork(2, 0, 260)          # a page that ends inside: its codes and scales are copied
    hk, hv = (held_fp8(x[0])[0] for x in (k, v))
    q = rows.normal(3, 4, 128)
    got = fork.decode_shared(0, q, 0.1)
    for r, n in enumerate([300, 300, 260]):
        check(got[r], attend(q[r:r + 1], hk, hv, 0.1, n - 1)[0][0])
        assert torch.equal(fork.gather(0, r, n)[0].double(), hk[:n].transpose(0, 1))
    fork.reorder([0, 1, 2], [2, 2, 0])
    for r, n in enumerate([260, 260, 300]):
        assert torch.equal(fork.gather(0, r, n)[1].double(), hv[:n].transpose(0, 1))


def test_step_in_one_call_equals_its_parts(sa):
    D, Hq, Hkv, lens = 128, 8, 2, [0, 63, 500]
    w = [1 + 0.1 * torch.randn(D, device="cuda") for _ in range(2)]
    rope = sa.rope_tables(1024, D)
    a, b = (Rows(sa, "fp8", Hkv, D, lens, seed=7, room=1) for _ in range(2))
    q, k, v = a.normal(3, Hq, D), a.normal(3, Hkv, D), a.normal(3, Hkv, D)
    q_out = torch.empty_like(q)
    one = a.cache.append_decode(0, q, k, v, 0.1, *w, rope=rope, q_out=q_out, commit=True)
    qn = b.cache.append(0, q[:, None], k[:, None], v[:, None], *w, rope=rope)[:, 0]
    b.cache.commit(1, n_seqs=3)
    two = b.cache.decode(0, qn.contiguous(), 0.1)
    assert torch.equal(q_out, qn) and torch.equal(one, two)
    plain = Rows(sa, "fp8", Hkv, D, lens, seed=7, room=1)
    assert torch.equal(plain.cache.append_decode(0, q, k, v, 0.1, *w, rope=rope), one)
    for r, n in enumerate(lens):
        assert a.cache.length(r) == n + 1 and plain.cache.length(r) == n
        for x, y in zip(a.cache.gather(0, r, n + 1), b.cache.gather(0, r, n + 1)):
            assert torch.equal(x, y)


def test_values_that_are_not_finite(sa):
    """A NaN in sight is one in the output; rows without one keep theirs."""
    def change(k, v):
        v[150, 0, 3] = float("inf")      # row 1, token 50; held as NaN
    rows = Rows(sa, "fp8", 1, 128, [100, 0, 100], seed=8, room=200)
    rows.append([0, 100, 0], commit=True)
    rows.append([0, 100, 0], commit=True, change=lambda k, v: v.__setitem__((50, 0, 3), float("inf")))
    q = rows.normal(3, 2, 128)
    got = rows.cache.decode(0, q, 0.1)
    assert got[1, :, 3].isnan().all() and got[1, :, :3].isfinite().all() and got[1, :, 4:].isfinite().all()
    for r in (0, 2):
        check(got[r], attend(q[r:r + 1], rows.k[r], rows.v[r], 0.1, 99)[0][0])


def test_scales_far_apart(sa):
    """Rows of very different magnitudes: values near 2^60 and 2^-60 in one sequence, keys whose scores stay small."""
    def change(k, v):
        v *= torch.exp2(torch.where(torch.arange(len(v), device="cuda") % 2 == 0, 60.0, -60.0))[:, None, None]
        k *= 2.0 ** -40
    rows = Rows(sa, "fp8", 1, 64, [0], seed=9, room=200)
    rows.append([200], commit=True, change=change)
    q = rows.normal(1, 1, 64) * 2.0 ** 40
    got = rows.cache.decode(0, q, 0.125)
    want = attend(q, rows.k[0], rows.v[0], 0.125, 199)[0]
    check(got / 2.0 ** 60, want / 2.0 ** 60)


def test_refusals(sa):
    for D in (8, 16, 32, 256):
        with pytest.raises(sa.SaError, match="8 bits take head_dim"):
            sa.KVCache(1, 1, D, 1, 1, 1, sa.SA_DTYPE_FP8)
    with pytest.raises(sa.SaError, match="kv_dtype"):
        sa.KVCache(1, 1, 64, 1, 1, 1, 3)
    cache = sa.KVCache(1, 1, 64, 1, 1, 1, sa.SA_DTYPE_F32)
    with pytest.raises(ValueError, match="scales"):
        sa.kv_scale_views(cache, 0)
    assert sa.lib().sa_kvcache_k_scales(cache.handle, 0) is None
    cache = sa.KVCache(2, 1, 64, 1, 1, 1, sa.SA_DTYPE_FP8)
    assert cache.nbytes() == 2 * 2 * 64 * 65
    assert sa.lib().sa_kvcache_v_scales(cache.handle, 2) is None
    cache.reserve(0, 64)
    cache.set_len(0, 64)
    q = torch.zeros(1, 65, 64, device="cuda")
    with pytest.raises(sa.SaError, match="64 query heads"):
        cache.decode(0, q, 1.0)
    with pytest.raises(sa.SaError, match="exceeds"):
        cache.decode(0, q[:, :1].contiguous(), 1.0, n_pending=1)
    k = torch.zeros(1, 1, 64, device="cuda")
    with pytest.raises(sa.SaError, match="full"):
        cache.append_decode(0, q[:, :1].contiguous(), k, k, 1.0)
    cache.set_len(0, 3)
    with pytest.raises(sa.SaError, match="workspace"):
        cache.append_decode(0, q[:, :1].contiguous(), k, k, 1.0, ws=torch.empty(16, dtype=torch.uint8, device="cuda"))
