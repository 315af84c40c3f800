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
