"""CPU checks of the largest calls: sizes whose launch would not fit a grid are
refused before anything touches a device, by the C entries themselves."""
from __future__ import annotations

import ctypes as C

import pytest

from util import load_pkg


@pytest.fixture(scope="module")
def sa():
    pkg = load_pkg()
    yield pkg
    pkg.lib().sa_prefill_window(None, None, None, pkg.SA_DTYPE_F32, 1, 1, 1, 0, 64, None, None, None, 1, 0, 1.0, None,
                                None)   # nothing to do: leaves no error behind


def test_prefill_window_grid(sa):
    """A grid has fewer than 2^32 threads: 2^23 workgroups of 512."""
    buf = (C.c_uint8 * 64)()
    at = (C.addressof(buf) + 15) // 16 * 16

    def call(B, Hq, L, window=1):
        return sa.lib().sa_prefill_window(at, at, at, sa.SA_DTYPE_BF16, B, Hq, 1, L, 64, None, None, None, window, 0,
                                          1.0, at, None)

    # 8 heads of one KV head: workgroups of 32 queries
    for B, Hq, L in ((1, 8, 1 << 30), (1 << 10, 8, 1 << 18), (1 << 23, 8, 1)):
        assert call(B, Hq, L) == sa.SA_EINVAL, (B, Hq, L)
        assert b"query tiles" in sa.lib().sa_last_error()


def test_beam_select_grid(sa):
    buf = (C.c_uint8 * 64)()
    at = (C.addressof(buf) + 15) // 16 * 16

    def call(G, B, V):
        return sa.lib().sa_beam_select(at, V, at, G, B, V, 1, at, at, at, at, 1 << 50, None)

    assert sa.beam_select_ws_bytes(1 << 20, 1, 5, 1) > 0 and sa.beam_select_ws_bytes((1 << 20) + 1, 1, 5, 1) == 0
    for G, B, V in (((1 << 20) + 1, 1, 5), (1 << 20, 16, 5), (1 << 14, 64, 40000)):
        assert call(G, B, V) == sa.SA_EINVAL, (G, B, V)
        assert sa.lib().sa_last_error()


def test_beam_search_arguments(sa):
    model = sa.Qwen3.__new__(sa.Qwen3)
    for beams, tokens in ((0, 5), (65, 5), (4, 0), (4, -1)):
        with pytest.raises(ValueError):
            model.beam_search(None, None, beams, tokens)


def test_beam_searches_that_cannot_end(sa):
    """More beams than the model's rows, or more tokens than its positions or the
    cache's pages: refused with the cache untouched."""
    import torch

    class Cache:
        desc = sa.KvDesc(1, 1, 64, 16, 4, 64, sa.SA_DTYPE_F32)

        def __getattr__(self, name):
            raise RuntimeError(f"the cache was touched: {name}")

    model = sa.Qwen3.__new__(sa.Qwen3)
    model.handle, model.max_batch = None, 8
    for max_pos, G, L, B, n, why in ((1000, 2, 10, 5, 3, "rows"), (1000, 3, 10, 6, 3, "row per beam"),
                                     (50, 1, 30, 4, 22, "positions"), (1000, 1, 200, 4, 58, "pages"),
                                     (300, 1, 300, 1, 1, "pages")):
        model.desc = sa.Qwen3Desc(1, 64, 64, 64, 1, 1, 64, max_pos, 1e-6, 1e6)
        for eos in (None, 3):
            with pytest.raises(ValueError, match=why):
                model.beam_search(Cache(), torch.zeros(G, L, dtype=torch.int32), B, n, eos)
    for max_pos, L, n in ((51, 30, 22), (1000, 200, 57)):       # the last that fit reach the cache
        model.desc = sa.Qwen3Desc(1, 64, 64, 64, 1, 1, 64, max_pos, 1e-6, 1e6)
        with pytest.raises(RuntimeError, match="touched"):
            model.beam_search(Cache(), torch.zeros(1, L, dtype=torch.int32), 4, n)


def test_scores_in_place_where_searches_would_meet(sa):
    """Searches run side by side: results of one may not fall on scores that
    another has yet to read.  (A workspace too small is what the calls that may
    run in place are refused for.)"""
    buf = (C.c_uint8 * 4096)()
    at = (C.addressof(buf) + 15) // 16 * 16
    model = (C.c_uint8 * 4096)()                # no call reads it
    far = at + 2048

    def select(G, B, n, scores, out):
        return sa.lib().sa_beam_select(at, 50, scores, G, B, 50, n, out, far, far + 512, far + 1024, 8, None)

    def step(G, B, n, scores, out):
        return sa.lib().sa_qwen3_beam_step(C.addressof(model), at, at, G, B, scores, n, out, far, far + 512, None)

    for call in (select, step):
        for G, B, n, shift in ((2, 2, 4, 0), (2, 4, 2, 0), (3, 1, 2, 0), (2, 4, 4, 4), (2, 4, 4, -4), (2, 2, 8, -60),
                               (1, 4, 4, 4), (1, 4, 8, -28), (3, 4, 4, 44)):
            assert call(G, B, n, at + 256, at + 256 + shift) == sa.SA_EINVAL, (call, G, B, n, shift)
            assert b"out_scores" in sa.lib().sa_last_error()
    for G, B, n, shift in ((2, 4, 4, 0), (1, 2, 4, 0), (1, 4, 2, 0), (2, 4, 2, 32), (2, 4, 8, -64), (1, 4, 4, 16)):
        assert select(G, B, n, at + 256, at + 256 + shift) == sa.SA_ENOMEM, (G, B, n, shift)
