"""GPU tests of forked and reordered sequences: the cached keys and values of
every row are bit for bit what the rows they came from held, appends go to
pages of the row's own, the device's table and lengths follow the host's, and
refused calls change nothing."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def gathered(cache, layer, row):
    n = cache.length(row)
    return torch.stack(cache.gather(layer, row, n)) if n else None


def device_table(sa, cache):
    """The device's block table and lengths."""
    d = cache.desc
    ptrs = (sa.lib().sa_kvcache_block_table(cache.handle), sa.lib().sa_kvcache_seq_lens(cache.handle))
    sizes = (d.max_seqs * d.max_pages_per_seq, d.max_seqs)
    torch.cuda.synchronize()
    views = [sa._device_view(p, n, torch.float32).view(torch.int32).cpu().numpy() for p, n in zip(ptrs, sizes)]
    return views[0].reshape(d.max_seqs, d.max_pages_per_seq), views[1]


def append(cache, layers, row, n, seed, Hkv, D):
    cache.reserve(row, cache.length(row) + n)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    for layer in range(layers):
        k, v = (torch.randn(1, n, Hkv, D, device="cuda", generator=gen) for _ in range(2))
        cache.append(layer, None, k, v, seq_ids=[row])
    cache.commit(n, seqs=[row])


@pytest.mark.parametrize("dtype,D", [("f32", 8), ("f32", 128), ("bf16", 8), ("bf16", 64), ("bf16", 256)])
@pytest.mark.parametrize("n", [1, 63, 64, 100, 128, 150])
def test_fork(sa, dtype, D, n):
    layers, Hkv = 2, 3
    cache = sa.KVCache(layers, Hkv, D, 3, 4, 10, sa.SA_DTYPE_BF16 if dtype == "bf16" else sa.SA_DTYPE_F32)
    append(cache, layers, 1, 150, 1, Hkv, D)
    append(cache, layers, 2, 70, 2, Hkv, D)      # what the fork replaces
    want = [gathered(cache, layer, 1) for layer in range(layers)]
    cache.fork(2, 1, n)
    cache.fork(0, 2, n // 2)
    assert [cache.length(r) for r in range(3)] == [n // 2, 150, n]
    for layer in range(layers):
        assert torch.equal(gathered(cache, layer, 2), want[layer][:, :, :n])
        if n > 1:
            assert torch.equal(gathered(cache, layer, 0), want[layer][:, :, :n // 2])
    # rows go on by themselves
    append(cache, layers, 2, 5, 3, Hkv, D)
    append(cache, layers, 1, 7, 4, Hkv, D)
    append(cache, layers, 0, 66, 5, Hkv, D)
    for layer in range(layers):
        for row, m in ((0, n // 2), (1, 150), (2, n)):
            if m:
                assert torch.equal(gathered(cache, layer, row)[:, :, :m], want[layer][:, :, :m]), row
    table, lens = device_table(sa, cache)
    assert list(lens) == [n // 2 + 66, 157, n + 5]
    assert (table[0, :(n // 2 + 66 + 63) // 64] >= 0).all() and (table[0, (n // 2 + 66 + 63) // 64:] == -1).all()
    cache.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("parents", [[0, 0, 0, 0, 0], [1, 2, 3, 4, 0], [0, 0, 3, 2, 2], [4, 1, 1, 1, 5], [0, 1, 2, 3, 4]])
def test_reorder(sa, dtype, parents):
    layers, Hkv, D = 3, 2, 64
    cache = sa.KVCache(layers, Hkv, D, 6, 6, 36, sa.SA_DTYPE_BF16 if dtype == "bf16" else sa.SA_DTYPE_F32)
    append(cache, layers, 0, 130, 10, Hkv, D)
    for r in range(1, 6):
        cache.fork(r, 0, 100 + 10 * (r % 3))
    for step in range(3):
        for r in range(6):
            append(cache, layers, r, 1 + (r + step) % 2 + 30 * (r == 3), 100 + 6 * step + r, Hkv, D)
        want = [[gathered(cache, layer, r) for r in range(6)] for layer in range(layers)]
        cache.reorder(range(5), parents)
        for layer in range(layers):
            for r in range(6):
                src = parents[r] if r < 5 else r
                assert torch.equal(gathered(cache, layer, r), want[layer][src]), (step, layer, r)
    table, lens = device_table(sa, cache)
    assert list(lens) == [cache.length(r) for r in range(6)]
    cache.close()


def test_reorder_of_many_rows_and_entries(sa):
    """More rows than one launch publishes, and more table entries."""
    layers, Hkv, D, rows = 1, 1, 8, 150
    cache = sa.KVCache(layers, Hkv, D, rows, 8, rows * 8)
    gen = torch.Generator(device="cuda").manual_seed(7)
    for r in range(rows):
        n = 1 + 3 * r
        cache.reserve(r, n)
        cache.append(0, None, torch.randn(1, n, Hkv, D, device="cuda", generator=gen),
                     torch.randn(1, n, Hkv, D, device="cuda", generator=gen), seq_ids=[r])
        cache.commit(n, seqs=[r])
    want = [gathered(cache, 0, r) for r in range(rows)]
    parents = [(7 * r + 3) % rows for r in range(rows)]
    cache.reorder(range(rows), parents)
    for r in range(rows):
        assert torch.equal(gathered(cache, 0, r), want[parents[r]]), r
    cache.close()


def test_refusals_change_nothing(sa):
    cache = sa.KVCache(1, 2, 64, 3, 3, 5)
    append(cache, 1, 0, 150, 1, 2, 64)            # three of five pages
    append(cache, 1, 1, 70, 2, 2, 64)             # the other two
    before = [gathered(cache, 0, r) for r in (0, 1)]
    table, lens = device_table(sa, cache)
    lib, h = sa.lib(), cache.handle
    ints = lambda *v: (C.c_int32 * len(v))(*v)  # noqa: E731
    assert lib.sa_kvcache_fork(None, 0, 1, 0, None) == sa.SA_EINVAL
    assert lib.sa_kvcache_fork(h, 0, 0, 1, None) == sa.SA_EINVAL
    assert lib.sa_kvcache_fork(h, 2, 0, 151, None) == sa.SA_ERANGE
    assert lib.sa_kvcache_fork(h, 3, 0, 1, None) == sa.SA_ERANGE
    assert lib.sa_kvcache_fork(h, 2, -1, 1, None) == sa.SA_ERANGE
    assert lib.sa_kvcache_fork(h, 2, 0, 150, None) == sa.SA_EFULL
    assert b"full" in lib.sa_last_error()
    assert lib.sa_kvcache_reorder(h, ints(0, 0), ints(1, 1), 2, None) == sa.SA_EINVAL
    assert lib.sa_kvcache_reorder(h, ints(0, 3), ints(1, 1), 2, None) == sa.SA_ERANGE
    assert lib.sa_kvcache_reorder(h, ints(0, 1), ints(1, 3), 2, None) == sa.SA_ERANGE
    assert lib.sa_kvcache_reorder(h, None, ints(1, 1), 2, None) == sa.SA_EINVAL
    assert lib.sa_kvcache_reorder(h, ints(0), ints(1), -1, None) == sa.SA_EINVAL
    assert lib.sa_kvcache_reorder(h, ints(2), ints(0), 1, None) == sa.SA_EFULL
    assert lib.sa_kvcache_reorder(None, ints(2), ints(0), 1, None) == sa.SA_EINVAL
    table2, lens2 = device_table(sa, cache)
    assert np.array_equal(table, table2) and np.array_equal(lens, lens2)
    for r in (0, 1):
        assert torch.equal(gathered(cache, 0, r), before[r])
    # a length set back into shared pages: nothing is written there
    cache.fork(2, 0, 128)
    cache.set_len(2, 100)
    x = torch.randn(1, 1, 2, 64, device="cuda")
    with pytest.raises(sa.SaError, match="shares"):
        cache.append(0, None, x, x, seq_ids=[2])
    with pytest.raises(sa.SaError, match="shares"):
        cache.append_decode(0, x[0], x[0], x[0], 1.0, seq_ids=[2])
    with pytest.raises(sa.SaError, match="another"):
        cache.set_pages(1, [0])
    assert torch.equal(gathered(cache, 0, 0), before[0])
    cache.close()


def test_on_a_stream_of_the_callers(sa):
    """All calls on one stream that is not the current one are ordered on it."""
    cache = sa.KVCache(2, 2, 64, 4, 4, 16)
    append(cache, 2, 0, 200, 1, 2, 64)
    want = [gathered(cache, layer, 0) for layer in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    big = torch.randn(4096, 4096, device="cuda")
    with torch.cuda.stream(side):
        for _ in range(5):
            big = big @ big * 1e-3      # the side stream is busy when the calls are made
    cache.fork(1, 0, 190, stream=side)
    cache.reorder([2, 3, 0], [1, 0, 1], stream=side)
    with torch.cuda.stream(side):
        got = [[gathered(cache, layer, r) for r in range(4)] for layer in range(2)]
    torch.cuda.synchronize()
    for layer in range(2):
        for r, n in enumerate([190, 190, 190, 200]):
            assert torch.equal(got[layer][r], want[layer][:, :, :n]), (layer, r)
    cache.close()


@pytest.mark.parametrize("n,old", [(300 * 64, 0), (300 * 64 + 5, 400 * 64), (64, 350 * 64), (0, 200 * 64)])
def test_fork_of_many_pages(sa, n, old):
    """Tables of more entries than a launch's arguments hold; room is added to a
    forked row in two steps."""
    cache = sa.KVCache(1, 1, 8, 3, 420, 1260, sa.SA_DTYPE_BF16)
    cache.reserve(2, 310 * 64)
    cache.set_len(2, 310 * 64 - 9)
    cache.reserve(0, old)
    cache.fork(0, 2, n)
    shared, own = n // 64, (n + 63) // 64
    for more in (0, 1, 100):
        cache.reserve(0, (own + more) * 64)
        table, lens = device_table(sa, cache)
        assert lens.tolist() == [n, 0, 310 * 64 - 9]
        assert (table[0, :shared] == table[2, :shared]).all() and (table[0, own + more:] == -1).all()
        fresh = table[0, shared:own + more]
        assert (fresh >= 0).all() and len(set(fresh) | set(table[2, :310])) == len(fresh) + 310
        assert (table[1] == -1).all() and (table[2, 310:] == -1).all()
    cache.close()
